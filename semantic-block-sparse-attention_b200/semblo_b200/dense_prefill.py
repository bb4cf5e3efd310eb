"""Exact attention of packed prompts: the dense counterpart of the block-sparse prefill, for requests too short
for the index and for layers that are not sparse.

Documents of any lengths lie one behind the other (``cu_seqlens``) and do not see each other; scores may be
capped, biased by distance, limited to a local window, and a document may have a prefix that all its queries
see (an instruction read both ways, or attention sinks in front of a window).  The reference leaves these
layers to the engine's stock attention (semblo/vllm_plugin/model.py:1169-1269 dispatches away from them)."""
from __future__ import annotations

import torch

from . import _lib
from ._lib import check, device_scope, dtype_code, lib, overlaps, raw_stream, refuse_gradients, require_cuda
from .kv8_cache import HEAD_DIMS, _mask_arguments, _per_request, _row_arguments
from .paged_attention import PagedSparseAttentionResult

MAX_GROUP = 128              # query heads per KV head


def dense_prefill_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, cu_seqlens_q: torch.Tensor,
                            cu_seqlens_k: torch.Tensor | None = None, sm_scale: float, causal: bool = True,
                            window: int = 0, prefix_lens: torch.Tensor | None = None, softcap: float | None = None,
                            alibi_slopes: torch.Tensor | None = None, out: torch.Tensor | None = None,
                            return_logsumexp: bool = False) -> PagedSparseAttentionResult:
    """Attention of ``q`` [Tq, Hq, D] over ``k``, ``v`` [Tk, Hkv, D] (bf16 or fp16; any token and head strides that
    are multiples of 8 elements, others are copied).

    Document d holds queries cu_seqlens_q[d] ... cu_seqlens_q[d + 1] - 1 and keys of cu_seqlens_k (default: the
    same).  Its queries are its last positions: query i stands at p = Lk - Lq + i and sees key j if j <= p (and
    p - j < ``window``, where one is given) or j < prefix_lens[d]; without ``causal`` every key of the document.
    Scores are q . k sm_scale, then ``softcap`` tanh(score / softcap), then minus alibi_slopes[h] |p - j|.  A row that
    sees nothing gives 0 and a log-sum-exp of -inf.  Rows behind the last document and in front of the first are left as
    they were in a given ``out``, and are 0 without one; their log-sum-exp is -inf.  ``out`` must not overlap an input.

    Keys behind a document's end are never used, whatever they hold; K and V inside a document have to be finite.  (In
    bf16 under a cap up to 52 the weights run from 2^-92 to 2^60 before they are divided: V beyond 2^43 overflows there,
    and V below 2^-34 loses bits in rows whose scores are all at -cap.)  What is packed beside a document does not change
    its result, unless the call's number of tokens cuts its keys into other pieces: then the weights are rounded to 16
    bits against other references."""
    require_cuda(q, k, v, cu_seqlens_q, cu_seqlens_k, prefix_lens, alibi_slopes, out)
    refuse_gradients(q, k, v, out)
    if q.ndim != 3 or k.ndim != 3 or v.shape != k.shape:
        raise ValueError("q must have shape [Tq, Hq, D], k and v [Tk, Hkv, D]")
    tokens_q, hq, dim = q.shape
    tokens_k, hkv, kdim = k.shape
    dtype, device = q.dtype, q.device
    if dtype not in (torch.bfloat16, torch.float16) or k.dtype != dtype or v.dtype != dtype:
        raise ValueError("q, k and v must all be bf16 or all fp16")
    if kdim != dim:
        raise ValueError(f"the head dimensions of q ({dim}) and k ({kdim}) differ")
    if dim not in HEAD_DIMS:
        raise ValueError(f"the head dimension must be one of {HEAD_DIMS} (got {dim})")
    if hkv == 0 or hq == 0 or hq % hkv:
        raise ValueError(f"query heads ({hq}) must be a multiple of the KV heads ({hkv})")
    if hq // hkv > MAX_GROUP:
        raise ValueError(f"at most {MAX_GROUP} query heads per KV head (got {hq // hkv})")
    if cu_seqlens_q.ndim != 1 or cu_seqlens_q.shape[0] < 1:
        raise ValueError("cu_seqlens_q must hold one more value than there are documents")
    docs = cu_seqlens_q.shape[0] - 1
    if k.device != device or v.device != device or cu_seqlens_q.device != device:
        raise ValueError("q, k, v and cu_seqlens must be on one device")
    cu_q = _per_request("cu_seqlens_q", cu_seqlens_q, docs + 1)
    if cu_seqlens_k is None:
        cu_k = cu_q
    else:
        if cu_seqlens_k.device != device:
            raise ValueError("q, k, v and cu_seqlens must be on one device")
        cu_k = _per_request("cu_seqlens_k", cu_seqlens_k, docs + 1)
    window, softcap, prefix_lens, alibi_slopes = _mask_arguments(window, softcap, prefix_lens, alibi_slopes, docs, hq, device)
    if not causal and (window or prefix_lens is not None):
        raise ValueError("a window or a prefix needs the causal mask")
    (q, *q_rows), (k, *k_rows), (v, *v_rows) = _row_arguments(q), _row_arguments(k), _row_arguments(v)
    if not float(sm_scale) > 0.0:
        raise ValueError(f"sm_scale must be positive (got {sm_scale})")
    given = out is not None
    if not given:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype != dtype or out.device != device or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError("out must be contiguous, 16-byte aligned and have the shape, type and device of q")
    elif any(overlaps(out, x) for x in (q, k, v)):
        raise ValueError("out must not overlap q, k or v")
    lse = None
    if return_logsumexp:
        lse = q.new_empty((tokens_q, hq), dtype=torch.float32)
        if given:
            lse.fill_(float("-inf"))
    with device_scope(device):
        nbytes = lib().semblo_dense_prefill_workspace_bytes(tokens_q, tokens_k, hq, hkv, dim, docs, bool(causal), window,
                                                            prefix_lens is not None)
        if nbytes < 0:
            check(int(nbytes))
        # made for this call: a recorded graph keeps its own, and calls on two streams do not share one
        workspace = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        check(lib().semblo_dense_prefill(
            *q_rows, *k_rows, *v_rows, tokens_q, tokens_k, hq, hkv, dim, dtype_code(dtype, "prefill"), cu_q.data_ptr(),
            cu_k.data_ptr(), docs, bool(causal), window, None if prefix_lens is None else prefix_lens.data_ptr(), sm_scale, softcap,
            None if alibi_slopes is None else alibi_slopes.data_ptr(), out.data_ptr(), not given,
            None if lse is None else lse.data_ptr(), None if workspace is None else workspace.data_ptr(), nbytes,
            _lib.status_for(device).word.data_ptr(), raw_stream(device.index)))
    return PagedSparseAttentionResult(out, lse)
