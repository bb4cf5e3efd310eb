"""Workloads of the dense-request operators: rotary positions, attention of a prompt with masks and a
capped score, writing a paged K/V cache held in 8 bits, and attention of generated tokens over it.

``listed()`` are the cases that are timed, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes
what a serving loop has in hand, ``run`` is one pass: elementary torch operations in 32 bits when ``own``
is false, the package's operators when it is true.  ``exact`` evaluates the definitions in 64 bits."""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_PKG = str(Path(__file__).resolve().parent.parent / "semantic-block-sparse-attention_b200")
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_E4M3_MAX = 448.0
_BUDGET = 1 << 29            # elements of the largest score buffer the plain forms make


def _package():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)


# ---------------------------------------------------------------------------------- cases

def _rotary(name, tokens, hq, hkv, dim, rotary, layout, dtype, scaling, first, inverse=False):
    return dict(name=name, op="rotary", tokens=tokens, hq=hq, hkv=hkv, dim=dim, rotary=rotary, layout=layout,
                dtype=dtype, scaling=scaling, first=first, inverse=inverse)


def _prompt(name, tokens, docs, hq, hkv, dim, dtype, softcap, window, prefix, alibi, causal=True, past=0):
    return dict(name=name, op="prompt", tokens=tokens, docs=docs, hq=hq, hkv=hkv, dim=dim, dtype=dtype,
                softcap=softcap, window=window, prefix=prefix, alibi=alibi, causal=causal, past=past)


def _append(name, batch, tokens, past, hkv, dim, block, dtype):
    return dict(name=name, op="append", batch=batch, tokens=tokens, past=past, hkv=hkv, dim=dim, block=block,
                dtype=dtype)


def _decode(name, batch, length, queries, hq, hkv, dim, block, dtype, softcap, window, prefix, alibi):
    return dict(name=name, op="decode", batch=batch, length=length, queries=queries, hq=hq, hkv=hkv, dim=dim,
                block=block, dtype=dtype, softcap=softcap, window=window, prefix=prefix, alibi=alibi)


def listed():
    return [
        # one generated token of one request at the end of a 524288-token context
        _rotary("rotary_one_token", 1, 16, 4, 256, 256, "half", "bf16", "none", 524288),
        # one query chunk of the head-sharded layer near a million positions, frequencies scaled for it
        _rotary("rotary_chunk", 8192, 32, 8, 128, 128, "half", "bf16", "yarn", 1040384),
        # a whole 131072-token prompt of a layer that rotates a quarter of the head, pairs interleaved
        _rotary("rotary_prompt_partial", 131072, 16, 4, 256, 64, "interleaved", "bf16", "wavelength", 0),
        # a short question behind a shared instruction that sees itself whole
        _prompt("prompt_short_prefix", 197, 1, 8, 2, 64, "fp16", 0.0, 0, 37, False),
        # many requests' prompts packed into one call, of every length
        _prompt("prompt_documents", 8192, 23, 32, 8, 128, "bf16", 0.0, 0, 0, True),
        # a chunk of a longer prompt in a layer with capped scores and a local window
        _prompt("prompt_capped_window", 8192, 1, 32, 8, 128, "bf16", 50.0, 4096, 64, False, True, 8192),
        # a long dense prompt, below the length from which the block-sparse path takes over
        _prompt("prompt_long", 32768, 1, 16, 4, 256, "bf16", 0.0, 0, 0, False),
        # one token of each of 64 running requests, at any place of their last block
        _append("append_tokens", 64, 1, 8192, 8, 128, 256, "bf16"),
        # a 131072-token prompt written whole
        _append("append_prompt", 1, 131072, 0, 4, 256, 256, "bf16"),
        # one request just after its first block
        _decode("decode_short", 1, 513, 1, 8, 2, 128, 256, "bf16", 0.0, 0, 0, False),
        # a batch of requests of every length in a layer with capped scores
        _decode("decode_batch", 64, 16384, 1, 32, 8, 128, 16, "bf16", 30.0, 0, 0, False),
        # one request at 524288 tokens
        _decode("decode_long", 1, 524288, 1, 16, 4, 256, 256, "bf16", 0.0, 0, 0, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "prompt", "append", "decode"])
    if op == "rotary":
        dim = rng.choice([64, 80, 128, 256])
        hkv = rng.choice([1, 2, 4, 8])
        hq = hkv * rng.choice([1, 2, 4, 8])
        rotary = rng.choice([dim, dim, dim // 2, 32])
        # no more elements than the largest listed case: 131072 tokens x 20 heads x 256
        most = min(131072, 131072 * 20 * 256 // ((hq + hkv) * dim))
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        tokens = _log(rng, 1, most // 2 if dtype == "fp32" else most)
        return dict(op=op, tokens=tokens, hq=hq, hkv=hkv, dim=dim, rotary=rotary,
                    layout=rng.choice(["half", "interleaved"]), dtype=dtype,
                    scaling=rng.choice(["none", "linear", "ntk", "yarn", "wavelength"]),
                    first=rng.choice([0, _log(rng, 1, 1 << 20)]), inverse=rng.random() < 0.2)
    if op == "prompt":
        dim = rng.choice([64, 128, 128, 256])
        hkv = rng.choice([1, 2, 4, 8])
        hq = hkv * rng.choice([1, 2, 4, 7, 8])
        tokens = _log(rng, 1, 8192)
        past = rng.choice([0, 0, _log(rng, 1, 4096)])
        return dict(op=op, tokens=tokens, docs=min(tokens, _log(rng, 1, 48)), hq=hq, hkv=hkv, dim=dim,
                    dtype=rng.choice(["bf16", "bf16", "fp16"]), softcap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                    window=rng.choice([0, 0, _log(rng, 1, 4096)]), prefix=rng.choice([0, 0, _log(rng, 1, 512)]),
                    alibi=rng.random() < 0.25, causal=True, past=past)
    if op == "append":
        hkv, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
        batch = _log(rng, 1, 128)
        most = max(1, 131072 * 4 * 256 // (hkv * dim * batch))
        tokens = rng.choice([1, _log(rng, 1, min(most, 131072))])
        return dict(op=op, batch=batch, tokens=tokens, past=rng.choice([0, _log(rng, 1, 8192)]), hkv=hkv, dim=dim,
                    block=rng.choice([16, 32, 64, 128, 256]), dtype=rng.choice(["bf16", "fp16"]))
    hkv = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 128, 256])
    batch = _log(rng, 1, 96)
    most = min(262144, max(64, 524288 * 4 * 256 // (hkv * dim * batch)))
    return dict(op="decode", batch=batch, length=_log(rng, 1, most), queries=rng.choice([1, 1, 1, 2, 5]),
                hq=hkv * rng.choice([1, 2, 4, 5, 8, 16]), hkv=hkv, dim=dim, block=rng.choice([16, 32, 64, 128, 256]),
                dtype=rng.choice(["bf16", "fp16"]), softcap=rng.choice([0.0, 0.0, 30.0]),
                window=rng.choice([0, 0, _log(rng, 1, 8192)]), prefix=rng.choice([0, 0, _log(rng, 1, 256)]),
                alibi=rng.random() < 0.25)


# ---------------------------------------------------------------------------------- shared pieces

def _spread(total, parts, gen):
    """``total`` cut into ``parts`` lengths of at least one, from short to long as requests come."""
    w = torch.rand(parts, generator=gen).mul(2.5).exp()
    lens = (w / w.sum() * (total - parts)).floor().long() + 1
    lens[int(torch.randint(parts, (1,), generator=gen))] += total - int(lens.sum())
    return [int(x) for x in lens]


def _lengths(case):
    """Host lengths of the documents or requests of a case (the same for every seed: they fix the shapes)."""
    gen = torch.Generator().manual_seed(11)
    if case["op"] == "prompt":
        q = _spread(case["tokens"], case["docs"], gen)
        past = [0] * len(q)
        if case["past"]:
            past = [int(x) for x in torch.randint(1, case["past"] + 1, (len(q),), generator=gen)]
            past[0] = case["past"]
        return q, [a + b for a, b in zip(q, past)]
    if case["op"] == "append":
        b = case["batch"]
        if case["tokens"] == 1:
            new = [1] * b
        else:
            new = [int(x) for x in torch.randint(1, case["tokens"] + 1, (b,), generator=gen)]
            new[0] = case["tokens"]
        past = [int(x) for x in torch.randint(0, case["past"] + 1, (b,), generator=gen)]
        return new, past
    b = case["batch"]
    lens = [int(math.exp(float(u) * math.log(case["length"]))) for u in torch.rand(b, generator=gen)]
    lens = [max(1, min(case["length"], (x + case["length"]) // 2)) for x in lens]
    lens[0] = case["length"]
    return lens, None


def _starts(lens):
    out = [0]
    for x in lens:
        out.append(out[-1] + x)
    return out


def _slopes(hq, device):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / hq) for i in range(hq)], dtype=torch.float32, device=device)


def _visible_pairs(q_lens, k_lens, window, prefix, causal):
    total = 0
    for lq, lk in zip(q_lens, k_lens):
        if not causal:
            total += lq * lk
            continue
        p0 = lk - lq
        pre = min(prefix, lk)
        p = torch.arange(p0, lk, dtype=torch.int64)
        lo = (p - window + 1).clamp_min(0) if window else torch.zeros_like(p)
        below = (p + 1 - torch.maximum(lo, torch.full_like(lo, pre))).clamp_min(0)
        total += int(below.sum()) + pre * lq
    return total


def work(case):
    e = 4 if case.get("dtype") == "fp32" else 2
    op = case["op"]
    if op == "rotary":
        rows = case["tokens"] * (case["hq"] + case["hkv"])
        return {"bytes": 2 * rows * case["dim"] * e + 8 * case["tokens"], "flops": 3 * rows * case["rotary"]}
    if op == "prompt":
        q_lens, k_lens = _lengths(case)
        pairs = _visible_pairs(q_lens, k_lens, case["window"], case["prefix"], case["causal"])
        by = (2 * sum(q_lens) * case["hq"] + 2 * sum(k_lens) * case["hkv"]) * case["dim"] * e
        return {"bytes": by + 4 * sum(q_lens) * case["hq"], "flops": 4 * pairs * case["hq"] * case["dim"]}
    if op == "append":
        new, past = _lengths(case)
        n = sum(new) * case["hkv"] * case["dim"]
        heads = 2 * 4 * case["hkv"]
        blocks = sum((p + x + case["block"] - 1) // case["block"] - p // case["block"] for x, p in zip(new, past))
        return {"bytes": 2 * n * (e + 1) + heads * blocks, "flops": 4 * n}
    lens, _ = _lengths(case)
    seen = 0
    for x in lens:
        w = min(x, case["window"] + case["queries"] - 1) if case["window"] else x
        seen += min(x, w + min(case["prefix"], x))
    pairs = _visible_pairs([min(case["queries"], x) for x in lens], lens, case["window"], case["prefix"], True)
    by = 2 * seen * case["hkv"] * case["dim"] + 2 * case["batch"] * case["queries"] * case["hq"] * case["dim"] * e
    return {"bytes": by, "flops": 4 * pairs * case["hq"] * case["dim"]}


# ---------------------------------------------------------------------------------- inputs

_ROPE = dict(base=500000.0, factor=8.0, original=131072, low=1.0, high=4.0, fast=32.0, slow=1.0)


def _frequencies(rotary, scaling):
    """Inverse frequencies in 64 bits and the factor on cos and sin."""
    r = _ROPE
    i = torch.arange(0, rotary, 2, dtype=torch.float64)
    base = r["base"]
    if scaling == "ntk":
        base = base * r["factor"] ** (rotary / max(rotary - 2, 1))
    inv = base ** (-i / rotary)
    if scaling == "linear":
        return inv / r["factor"], 1.0
    if scaling == "yarn":
        def dim_of(turns):
            return rotary * math.log(r["original"] / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo = max(math.floor(dim_of(r["fast"])), 0)
        hi = min(math.ceil(dim_of(r["slow"])), rotary - 1)
        ramp = ((torch.arange(rotary // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return inv / r["factor"] * ramp + inv * (1 - ramp), 0.1 * math.log(r["factor"]) + 1.0
    if scaling == "wavelength":
        turns = r["original"] * inv / (2 * math.pi)
        keep = ((turns - r["low"]) / (r["high"] - r["low"])).clamp(0, 1)
        return inv * (keep + (1 - keep) / r["factor"]), 1.0
    return inv, 1.0


def _scaling_spec(scaling):
    r = _ROPE
    if scaling == "none":
        return None
    spec = {"type": scaling, "factor": r["factor"]}
    if scaling == "yarn":
        spec.update(original_max_position=r["original"], beta_fast=r["fast"], beta_slow=r["slow"])
    if scaling == "wavelength":
        spec.update(original_max_position=r["original"], low_freq_factor=r["low"], high_freq_factor=r["high"])
    return spec


def _normal(gen, *shape, dtype, scale=1.0):
    x = torch.empty(*shape, dtype=dtype, device="cuda")
    return x.normal_(0.0, scale, generator=gen)


def _need(amax):
    """The power of two that a block of largest magnitude ``amax`` is divided by, so that it stays below 448."""
    m, e = torch.frexp(amax)
    e = torch.where(m > 0.875, e - 8, e - 9)
    e = torch.where(amax > 0, e, torch.full_like(e, -100)).clamp(-100, 120)
    return torch.ldexp(torch.ones_like(amax), e)


def _to_e4m3(x):
    return x.clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn)


def _filled_cache(gen, blocks, block, hkv, dim):
    """A pool of written blocks [2, blocks, heads, tokens, dim]: normal keys and values, in steps of the
    block's own magnitude."""
    data = torch.empty(2, blocks, hkv, block, dim, dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty(2, blocks, hkv, dtype=torch.float32, device="cuda")
    step = max(1, (1 << 27) // (block * hkv * dim))
    for part in range(2):
        for i in range(0, blocks, step):
            n = min(step, blocks - i)
            x = _normal(gen, n, hkv, block, dim, dtype=torch.float32)
            x *= torch.exp2(torch.randint(-2, 3, (n, hkv, 1, 1), device="cuda", generator=gen).float() / 2)
            s = _need(x.abs().amax(dim=(2, 3)))
            data[part, i:i + n] = _to_e4m3(x / s[..., None, None])
            scales[part, i:i + n] = s
    return data, scales


def _table(gen, lens, block, spare=1):
    """A block table over a pool in random order; entries past a request's blocks hold 0."""
    need = [max(1, -(-x // block)) for x in lens]
    blocks = sum(need) + spare
    order = torch.randperm(blocks, device="cuda", generator=gen, dtype=torch.int64).to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, blocks


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 104729 + 3)
    dt = _DTYPES[case["dtype"]]
    op = case["op"]
    st = dict(case=case)
    if op == "rotary":
        t, d = case["tokens"], case["dim"]
        # q and k as the fused projection leaves them: heads of one token side by side
        qkv = _normal(gen, t, case["hq"] + 2 * case["hkv"], d, dtype=dt)
        st["q"], st["k"] = qkv[:, :case["hq"]], qkv[:, case["hq"]:case["hq"] + case["hkv"]]
        st["positions"] = torch.arange(case["first"], case["first"] + t, dtype=torch.int64, device="cuda")
        if own:
            _package()
            from semblo_b200.rotary import rotary_frequencies
            st["plan"] = rotary_frequencies(case["rotary"], _ROPE["base"], scaling=_scaling_spec(case["scaling"]),
                                            device="cuda")
        else:
            inv, scale = _frequencies(case["rotary"], case["scaling"])
            st["inv_freq"], st["scale"] = inv.cuda(), scale
        return st
    hq, hkv, d = case.get("hq"), case["hkv"], case["dim"]
    if op == "prompt":
        st["q_lens"], st["k_lens"] = _lengths(case)
        st["cu_q"] = torch.tensor(_starts(st["q_lens"]), dtype=torch.int32, device="cuda")
        st["cu_k"] = torch.tensor(_starts(st["k_lens"]), dtype=torch.int32, device="cuda")
        st["q"] = _normal(gen, sum(st["q_lens"]), hq, d, dtype=dt, scale=6.0 if case["softcap"] else 2.0)
        st["k"] = _normal(gen, sum(st["k_lens"]), hkv, d, dtype=dt)
        st["v"] = _normal(gen, sum(st["k_lens"]), hkv, d, dtype=dt)
        st["prefix"] = [min(case["prefix"], x) for x in st["k_lens"]]
        st["prefix_t"] = torch.tensor(st["prefix"], dtype=torch.int32, device="cuda") if case["prefix"] else None
        st["slopes"] = _slopes(hq, "cuda") if case["alibi"] else None
        return st
    if op == "append":
        st["new"], st["past"] = _lengths(case)
        after = [a + b for a, b in zip(st["new"], st["past"])]
        st["table"], blocks = _table(gen, after, case["block"])
        st["data"], st["scales"] = _filled_cache(gen, blocks, case["block"], hkv, d)
        st["cu"] = torch.tensor(_starts(st["new"]), dtype=torch.int32, device="cuda")
        st["start"] = torch.tensor(st["past"], dtype=torch.int32, device="cuda")
        n = sum(st["new"])
        lift = torch.exp2(torch.randint(-2, 4, (n, 1, 1), device="cuda", generator=gen).float() / 2)
        st["k"] = _normal(gen, n, hkv, d, dtype=dt).mul_(lift)
        st["v"] = _normal(gen, n, hkv, d, dtype=dt).mul_(lift)
    else:
        st["lens"], _ = _lengths(case)
        st["table"], blocks = _table(gen, st["lens"], case["block"])
        st["data"], st["scales"] = _filled_cache(gen, blocks, case["block"], hkv, d)
        st["lengths"] = torch.tensor(st["lens"], dtype=torch.int32, device="cuda")
        st["q"] = _normal(gen, case["batch"], case["queries"], hq, d, dtype=dt,
                          scale=6.0 if case["softcap"] else 3.0)
        st["prefix"] = [min(case["prefix"], x) for x in st["lens"]]
        st["prefix_t"] = torch.tensor(st["prefix"], dtype=torch.int32, device="cuda") if case["prefix"] else None
        st["slopes"] = _slopes(hq, "cuda") if case["alibi"] else None
    if own:
        _package()
        from semblo_b200.kv8_cache import Kv8Cache
        st["cache"] = Kv8Cache(st["data"], st["scales"])
    return st


# ---------------------------------------------------------------------------------- plain forms

def _plain_rotate(x, cos, sin, rotary, layout):
    y = x.float().clone()
    if layout == "half":
        a, b = y[..., :rotary // 2], y[..., rotary // 2:rotary]
    else:
        a, b = y[..., 0:rotary:2], y[..., 1:rotary:2]
    na, nb = a * cos - b * sin, b * cos + a * sin
    a.copy_(na)
    b.copy_(nb)
    return y.to(x.dtype)


def _plain_rotary(st):
    c = st["case"]
    angle = st["positions"].double()[:, None] * st["inv_freq"]
    cos = (angle.cos() * st["scale"]).float()[:, None]
    sin = (angle.sin() * st["scale"]).float()[:, None]
    if c["inverse"]:
        sin = -sin
    return [_plain_rotate(st[n], cos, sin, c["rotary"], c["layout"]) for n in ("q", "k")]


def _plain_attend(q, k, v, first, c, prefix, slopes):
    """q [Lq, Hq, D] at positions first ..., k and v [Lk, Hkv, D], all in 32 bits -> output, log-sum-exp."""
    lq, hq, d = q.shape
    lk, hkv, _ = k.shape
    g = hq // hkv
    out = torch.zeros(lq, hq, d, dtype=torch.float32, device=q.device)
    lse = torch.full((lq, hq), -math.inf, dtype=torch.float32, device=q.device)
    if lk == 0 or lq == 0:
        return out, lse
    kt = k.permute(1, 2, 0)
    vt = v.permute(1, 0, 2)
    j = torch.arange(lk, device=q.device)
    step = max(1, _BUDGET // (hq * lk))
    for i in range(0, lq, step):
        n = min(step, lq - i)
        p = torch.arange(first + i, first + i + n, device=q.device)
        qs = q[i:i + n].reshape(n, hkv, g, d).permute(1, 2, 0, 3).reshape(hkv, g * n, d)
        s = torch.matmul(qs, kt).view(hkv, g, n, lk) * d ** -0.5
        if c["softcap"]:
            s = c["softcap"] * torch.tanh(s / c["softcap"])
        dist = p[:, None] - j[None, :]
        if slopes is not None:
            s = s - slopes.view(hkv, g, 1, 1) * dist.abs().float()
        if c.get("causal", True):
            see = dist >= 0
            if c["window"]:
                see &= dist < c["window"]
            if prefix:
                see |= (j < prefix)[None, :]
            s = s.masked_fill(~see, -math.inf)
        top = s.amax(dim=-1, keepdim=True)
        top = torch.where(top == -math.inf, torch.zeros_like(top), top)
        e = torch.exp(s - top)
        total = e.sum(dim=-1, keepdim=True)
        o = torch.matmul(e.view(hkv, g * n, lk), vt).view(hkv, g, n, d) / total.clamp_min(1e-37)
        out[i:i + n] = o.permute(2, 0, 1, 3).reshape(n, hq, d)
        lse[i:i + n] = (top + total.log()).squeeze(-1).permute(2, 0, 1).reshape(n, hq)
    return out, lse


def _plain_prompt(st):
    c = st["case"]
    q0, k0 = _starts(st["q_lens"]), _starts(st["k_lens"])
    out = torch.empty_like(st["q"])
    lse = torch.empty(st["q"].shape[:2], dtype=torch.float32, device=st["q"].device)
    for b, (lq, lk) in enumerate(zip(st["q_lens"], st["k_lens"])):
        k, v = st["k"][k0[b]:k0[b] + lk].float(), st["v"][k0[b]:k0[b] + lk].float()
        o, ls = _plain_attend(st["q"][q0[b]:q0[b] + lq].float(), k, v, lk - lq, c, st["prefix"][b], st["slopes"])
        out[q0[b]:q0[b] + lq] = o.to(out.dtype)
        lse[q0[b]:q0[b] + lq] = ls
    return out, lse


def _plain_append(st):
    c = st["case"]
    block, dev = c["block"], st["k"].device
    new, past = (torch.tensor(st[n], device=dev) for n in ("new", "past"))
    first = past // block
    blocks = (past + new + block - 1) // block - first           # blocks that each request touches
    pair0 = torch.cumsum(blocks, 0) - blocks
    owner = torch.repeat_interleave(torch.arange(len(st["new"]), device=dev), new)
    pos = past[owner] + torch.arange(owner.numel(), device=dev) - (torch.cumsum(new, 0) - new)[owner]
    pair, slot = pair0[owner] + pos // block - first[owner], pos % block
    who = torch.repeat_interleave(torch.arange(len(st["new"]), device=dev), blocks)
    nth = torch.arange(who.numel(), device=dev) - pair0[who]
    pages = st["table"][who, first[who] + nth].long()
    keep = torch.where(nth == 0, past[who] % block, torch.zeros_like(nth))      # rows written by earlier calls
    row = torch.arange(block, device=dev)
    for part, x in enumerate((st["k"], st["v"])):
        fresh = torch.zeros(pages.numel(), c["hkv"], block, c["dim"], dtype=torch.float32, device=dev)
        fresh[pair, :, slot] = x.float()
        before = st["scales"][part][pages]
        scale = _need(fresh.abs().amax(dim=(2, 3)))
        scale = torch.where((keep > 0)[:, None], torch.maximum(scale, before), scale)
        held = st["data"][part][pages]
        old = _to_e4m3(held.float() * (before / scale)[..., None, None])
        code = _to_e4m3(fresh / scale[..., None, None])
        code = torch.where((row < keep[:, None])[:, None, :, None], old.view(torch.uint8), code.view(torch.uint8))
        last = torch.minimum(past[who] + new[who] - (first[who] + nth) * block, torch.full_like(nth, block))
        code = torch.where((row < last[:, None])[:, None, :, None], code, held.view(torch.uint8))
        st["data"][part].view(torch.uint8)[pages] = code
        st["scales"][part][pages] = scale
    return st["data"], st["scales"]


def _plain_decode(st):
    c = st["case"]
    block = c["block"]
    outs, lses = [], []
    for b, n in enumerate(st["lens"]):
        pages = st["table"][b, :-(-n // block)].long()
        k, v = (st["data"][p][pages].float().mul_(st["scales"][p][pages][..., None, None])
                .transpose(1, 2).reshape(-1, c["hkv"], c["dim"])[:n] for p in range(2))
        o, ls = _plain_attend(st["q"][b].float(), k, v, n - c["queries"], c, st["prefix"][b], st["slopes"])
        outs.append(o.to(st["q"].dtype))
        lses.append(ls)
    return torch.stack(outs), torch.stack(lses)


# ---------------------------------------------------------------------------------- one pass

def run(state):
    op = state["case"]["op"]
    if not own:
        return {"rotary": _plain_rotary, "prompt": _plain_prompt, "append": _plain_append,
                "decode": _plain_decode}[op](state)
    c = state["case"]
    if op == "rotary":
        from semblo_b200.rotary import apply_rotary
        return list(apply_rotary(state["q"], state["k"], state["positions"], state["plan"],
                                 interleaved=c["layout"] == "interleaved", inverse=c["inverse"]))
    if op == "prompt":
        from semblo_b200.dense_prefill import dense_prefill_attention
        r = dense_prefill_attention(state["q"], state["k"], state["v"], cu_seqlens_q=state["cu_q"],
                                    cu_seqlens_k=state["cu_k"], sm_scale=c["dim"] ** -0.5, causal=c["causal"],
                                    window=c["window"], prefix_lens=state["prefix_t"], softcap=c["softcap"],
                                    alibi_slopes=state["slopes"], return_logsumexp=True)
        return r.output, r.logsumexp
    if op == "append":
        from semblo_b200.kv8_cache import kv8_append
        kv8_append(state["cache"], state["k"], state["v"], state["table"], state["cu"], state["start"])
        return state["cache"].data, state["cache"].scales
    from semblo_b200.kv8_cache import kv8_decode_attention
    r = kv8_decode_attention(state["q"], state["cache"], state["table"], state["lengths"],
                             sm_scale=c["dim"] ** -0.5, softcap=c["softcap"], window=c["window"],
                             prefix_lens=state["prefix_t"], alibi_slopes=state["slopes"], return_logsumexp=True)
    return r.output, r.logsumexp


# ---------------------------------------------------------------------------------- definitions in 64 bits

def _exact_rows(q, k, v, p, c, prefix, slope):
    """One head: q [n, D] at positions p [n], k and v [L, D], all in 64 bits."""
    n, d = q.shape
    s = q @ k.T / math.sqrt(d)
    if c["softcap"]:
        s = torch.tanh(s / c["softcap"]) * c["softcap"]
    j = torch.arange(k.shape[0], device=q.device)
    if slope is not None:
        s = s - float(slope) * (p[:, None] - j).abs()
    if c.get("causal", True):
        first = p - c["window"] + 1 if c["window"] else torch.zeros_like(p)
        hidden = (j > p[:, None]) | (j < first[:, None])
        hidden &= j >= prefix
        s[hidden] = -math.inf
    lse = torch.logsumexp(s, dim=1)
    w = torch.exp(s - torch.where(lse.isinf(), torch.zeros_like(lse), lse)[:, None])
    return w @ v, lse


def _exact_document(q, k, v, first, c, prefix, slopes):
    hq, hkv = q.shape[1], k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    step = max(1, (1 << 27) // max(1, k.shape[0]))
    for h in range(hq):
        kh, vh = k[:, h * hkv // hq].double(), v[:, h * hkv // hq].double()
        for i in range(0, q.shape[0], step):
            n = min(step, q.shape[0] - i)
            p = torch.arange(first + i, first + i + n, device=q.device)
            out[i:i + n, h], lse[i:i + n, h] = _exact_rows(q[i:i + n, h].double(), kh, vh, p, c, prefix,
                                                          None if slopes is None else slopes[h])
    return out, lse


def _exact_append(st):
    c = st["case"]
    block, cu = c["block"], _starts(st["new"])
    data, scales = st["data"].double(), st["scales"].double()
    table = st["table"].cpu()
    for part, x in enumerate((st["k"].double(), st["v"].double())):
        for b, (n, past) in enumerate(zip(st["new"], st["past"])):
            at = past
            while at < past + n:
                page, off = int(table[b, at // block]), at % block
                m = min(block - off, past + n - at)
                rows = x[cu[b] + at - past:cu[b] + at - past + m]
                top = rows.abs().amax(dim=(0, 2)) / _E4M3_MAX
                s = torch.where(top > 0, torch.exp2(torch.ceil(torch.log2(top.clamp_min(2.0 ** -100)))),
                                torch.full_like(top, 2.0 ** -100))
                # the logarithm's rounding must not move a whole power of two
                s = torch.where(top > s, s * 2, torch.where((top <= s / 2) & (s > 2.0 ** -100), s / 2, s))
                if off:
                    s = torch.maximum(s, scales[part, page])
                    old = data[part, page, :, :off] * (scales[part, page] / s)[:, None, None]
                    data[part, page, :, :off] = old.float().to(torch.float8_e4m3fn).double()
                data[part, page, :, off:off + m] = (rows / s[None, :, None]).clamp(-448, 448).float() \
                    .to(torch.float8_e4m3fn).double().transpose(0, 1)
                scales[part, page] = s
                at += m
    return data, scales


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "rotary":
        inv, scale = _frequencies(case["rotary"], case["scaling"])
        inv = inv.to(st["q"].device)
        r = case["rotary"]
        res = []
        for x in (st["q"], st["k"]):
            y = x.double()
            for i in range(r // 2):
                a, b = (i, i + r // 2) if case["layout"] == "half" else (2 * i, 2 * i + 1)
                w = st["positions"].double() * inv[i]
                z = torch.polar(torch.full_like(w, scale), -w if case["inverse"] else w)[:, None]
                turned = torch.complex(y[..., a].clone(), y[..., b].clone()) * z
                y[..., a], y[..., b] = turned.real, turned.imag
            res.append(y)
        return res
    if op == "append":
        if sum(-(-x // case["block"]) + 1 for x in st["new"]) > 12000:
            return None
        return _exact_append(st)
    if op == "prompt":
        outs, lses = [], []
        q0, k0 = _starts(st["q_lens"]), _starts(st["k_lens"])
        for b, (lq, lk) in enumerate(zip(st["q_lens"], st["k_lens"])):
            o, ls = _exact_document(st["q"][q0[b]:q0[b + 1]], st["k"][k0[b]:k0[b + 1]], st["v"][k0[b]:k0[b + 1]],
                                    lk - lq, case, st["prefix"][b], st["slopes"])
            outs.append(o)
            lses.append(ls)
        return torch.cat(outs), torch.cat(lses)
    outs, lses = [], []
    for b, n in enumerate(st["lens"]):
        pages = st["table"][b, :-(-n // case["block"])].long()
        k, v = ((st["data"][p][pages].double() * st["scales"][p][pages].double()[..., None, None])
                .transpose(1, 2).reshape(-1, case["hkv"], case["dim"])[:n] for p in range(2))
        o, ls = _exact_document(st["q"][b], k, v, n - case["queries"], case, st["prefix"][b], st["slopes"])
        outs.append(o)
        lses.append(ls)
    return torch.stack(outs), torch.stack(lses)
