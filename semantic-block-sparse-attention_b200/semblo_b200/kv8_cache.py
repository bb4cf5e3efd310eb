"""A paged K/V cache held in 8 bits with a scale for each block of tokens and KV head: the store, the
append that quantises into it, and the attention of generated tokens over it.

The bf16 stores of the sparse path (the cluster-ordered copy, the suffix store) hold what the index
selects from; this cache holds every token of a dense request in half the bytes.  Codes are e4m3
[2, blocks, Hkv, block, D]: the tokens of one (block, head) lie side by side, so the attention of a head
reads whole kilobytes where the token-major layout of the bf16 stores would give it pieces of D bytes.
The reference has no 8-bit store."""
from __future__ import annotations

import torch

from . import _lib
from ._lib import (check, device_scope, dtype_code, lib, overlaps, raw_stream, refuse_gradients, require_cuda,
                   require_same_device)
from .paged_attention import PagedSparseAttentionResult

BLOCK_SIZES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128, 256)


class Kv8Cache:
    """``data`` [2, blocks, Hkv, block, D] float8_e4m3fn (K, V) and ``scales`` [2, blocks, Hkv] fp32: a stored value
    is code * scale.  Any positive scales may be read; :func:`kv8_append` writes powers of two."""

    def __init__(self, data: torch.Tensor, scales: torch.Tensor) -> None:
        if data.ndim != 5 or data.shape[0] != 2 or data.dtype != torch.float8_e4m3fn or not data.is_contiguous():
            raise ValueError("the 8-bit cache is a contiguous float8_e4m3fn tensor [2, blocks, Hkv, block, D]")
        _, self.num_blocks, self.num_kv_heads, self.block_size, self.head_dim = (int(n) for n in data.shape)
        if scales.shape != (2, self.num_blocks, self.num_kv_heads) or scales.dtype != torch.float32 \
                or not scales.is_contiguous():
            raise ValueError("scales must be contiguous fp32 [2, blocks, Hkv]")
        if self.block_size not in BLOCK_SIZES:
            raise ValueError(f"the block size must be one of {BLOCK_SIZES} (got {self.block_size})")
        if self.head_dim not in HEAD_DIMS:
            raise ValueError(f"the head dimension must be one of {HEAD_DIMS} (got {self.head_dim})")
        if scales.device != data.device:
            raise ValueError("codes and scales must be on one device")
        self.data = data
        self.scales = scales

    @classmethod
    def allocate(cls, num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int, device="cuda") -> "Kv8Cache":
        """An empty pool (a block's scale is set by the first call that writes it)."""
        shape = (2, int(num_blocks), int(num_kv_heads), int(block_size), int(head_dim))
        data = torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        return cls(data, torch.ones(shape[:3], dtype=torch.float32, device=device))

    def gather(self, pages: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """K and V of the listed blocks as fp32 [len(pages) * block, Hkv, D] (for inspection)."""
        pages = pages.long()
        out = []
        for part in range(2):
            x = self.data[part][pages].float() * self.scales[part][pages][..., None, None]
            out.append(x.transpose(1, 2).reshape(-1, self.num_kv_heads, self.head_dim))
        return out[0], out[1]


def _narrowed(x: torch.Tensor) -> torch.Tensor:
    """64-bit values as the kernels' 32-bit ones: those that do not fit stay out of every range."""
    return x.clamp(-(1 << 31), (1 << 31) - 1).to(torch.int32)


def _block_table(table: torch.Tensor, batch: int) -> torch.Tensor:
    if table.ndim != 2 or int(table.shape[0]) != batch:
        raise ValueError(f"the block table must have shape [{batch}, blocks per request] (got {tuple(table.shape)})")
    if table.dtype == torch.int64:
        table = _narrowed(table)
    elif table.dtype != torch.int32:
        if table.dtype not in (torch.int16, torch.int8, torch.uint8):
            raise ValueError(f"the block table must be whole numbers (got {table.dtype})")
        table = table.to(torch.int32)
    return table if table.stride(1) == 1 or table.shape[1] <= 1 else table.contiguous()


def _per_request(name: str, x: torch.Tensor, n: int) -> torch.Tensor:
    if x.shape != (n,) or x.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be {n} int32 or int64 values (got {x.dtype} {tuple(x.shape)})")
    if x.dtype != torch.int32:
        x = _narrowed(x)
    return x if x.is_contiguous() else x.contiguous()


def _token_rows(x: torch.Tensor) -> torch.Tensor:
    """x [T, H, D] as the kernels read it: contiguous heads of a 16-byte aligned start and step."""
    return _row_arguments(x)[0]


def _row_arguments(x: torch.Tensor) -> tuple:
    """(the rows as the kernels read them, their address, token stride, head stride)"""
    s0, s1, s2 = x.stride()
    address = x.data_ptr()
    if s2 != 1 or (address | 2 * s0 | 2 * s1) & 15 or s0 <= 0 or s1 <= 0:
        x = x.clone(memory_format=torch.contiguous_format)
        address = x.data_ptr()
        s0, s1, _ = x.stride()
    return x, address, s0, s1


def kv8_append(cache: Kv8Cache, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, cu_seqlens: torch.Tensor,
               start_positions: torch.Tensor) -> None:
    """Write ``k``, ``v`` [T, Hkv, D] (bf16 or fp16) into the cache.

    Tokens cu_seqlens[b] ... cu_seqlens[b + 1] - 1 are positions start_positions[b], start_positions[b] + 1, ... of
    request b and go to block ``block_table[b, position // block]``.  A block that starts with this call takes the
    smallest power-of-two scale that holds its largest finite magnitude; one that is continued keeps its scale
    unless a new value needs a larger one, and then the rows already there follow.  Infinities saturate, NaN stay
    NaN.  Rows of ``k`` / ``v`` behind the last request and rows of a block behind the last token are left as they
    are.  Two requests of one call must not share a block they write, and ``k`` and
    ``v`` must lie apart from the cache.  A table entry outside the pool, a position
    outside the table or a negative start sets status 201, and what it names is not written."""
    require_cuda(cache.data, k, v, block_table, cu_seqlens, start_positions)
    refuse_gradients(k, v)
    shape = tuple(k.shape)
    if len(shape) != 3 or shape[1:] != (cache.num_kv_heads, cache.head_dim) or tuple(v.shape) != shape:
        raise ValueError(f"k and v must have shape [T, {cache.num_kv_heads}, {cache.head_dim}] "
                         f"(got {shape} and {tuple(v.shape)})")
    if k.dtype != v.dtype or k.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("k and v must both be bf16 or both fp16")
    if cu_seqlens.ndim != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError("cu_seqlens must hold one more value than there are requests")
    batch = int(cu_seqlens.shape[0]) - 1
    require_same_device(cache.data, k, v, block_table, cu_seqlens, start_positions)
    table = _block_table(block_table, batch)
    cu, start = _per_request("cu_seqlens", cu_seqlens, batch + 1), _per_request("start_positions", start_positions, batch)
    (k, *k_rows), (v, *v_rows) = _row_arguments(k), _row_arguments(v)
    device = k.device
    with device_scope(device):
        check(lib().semblo_kv8_append(
            *k_rows, *v_rows, shape[0],
            dtype_code(k.dtype, "append"), cache.data.data_ptr(), cache.scales.data_ptr(), cache.num_blocks,
            cache.block_size, cache.num_kv_heads, cache.head_dim, table.data_ptr(), table.stride(0), table.shape[1],
            cu.data_ptr(), start.data_ptr(), batch, _lib.status_for(device).word.data_ptr(),
            raw_stream(device.index)))


MAX_QUERIES = 16
MIN_CAP, MAX_CAP = 2.0 ** -100, 2.0 ** 100       # so that neither the cap nor what divides a score by it leaves 32 bits


def _mask_arguments(window, softcap, prefix_lens, alibi_slopes, batch: int, heads: int, device):
    """The masks and caps that the dense operators share, checked: (window, softcap, prefix, slopes)."""
    window = int(window or 0)
    if window < 0:
        raise ValueError(f"the window must not be negative (got {window}; 0 is none)")
    window = min(window, 1 << 30)            # beyond every position, and inside the kernels' arithmetic
    softcap = float(softcap or 0.0)
    if softcap != 0.0 and not MIN_CAP <= softcap <= MAX_CAP:
        raise ValueError(f"the soft cap must lie in [2^-100, 2^100] (got {softcap}; 0 is none)")
    if prefix_lens is not None:
        prefix_lens = _per_request("prefix_lens", prefix_lens, batch)
        if prefix_lens.device != device:
            raise ValueError("prefix_lens must be on the device of the queries")
    if alibi_slopes is not None:
        if alibi_slopes.shape != (heads,) or alibi_slopes.dtype != torch.float32:
            raise ValueError(f"alibi_slopes must be {heads} fp32 values, one for each query head")
        if alibi_slopes.device != device:
            raise ValueError("alibi_slopes must be on the device of the queries")
        alibi_slopes = alibi_slopes.contiguous()
    return window, softcap, prefix_lens, alibi_slopes


def kv8_decode_attention(q: torch.Tensor, cache: Kv8Cache, block_table: torch.Tensor, lengths: torch.Tensor, *,
                         sm_scale: float, softcap: float | None = None, window: int = 0,
                         prefix_lens: torch.Tensor | None = None, alibi_slopes: torch.Tensor | None = None,
                         out: torch.Tensor | None = None, return_logsumexp: bool = False) -> PagedSparseAttentionResult:
    """Attention of the last tokens of each request (up to 4096 of them) over the 8-bit cache.

    ``q`` [B, n, Hq, D] (bf16 or fp16; 1 to 16 queries per request): query i of request b stands at position
    p = lengths[b] - n + i and sees key j < lengths[b] if j <= p (and p - j < ``window``, where one is given) or
    j < prefix_lens[b].  Scores are q . k sm_scale, then ``softcap`` tanh(score / softcap), then minus
    alibi_slopes[h] |p - j|.  A row that sees nothing (a length of 0, a position below 0) gives 0 and a log-sum-exp
    of -inf.  Keys that no query of a request sees may hold anything; a NaN in the V of a key that one of them sees
    reaches all of them.  The result [B, n, Hq, D] (``out``, apart from the
    inputs, where it is given) has the type of ``q``; log-sum-exps are natural, fp32 [B, n, Hq].  Table
    entries outside the pool are taken as absent and set status 201, as does a length beyond the table."""
    require_cuda(q, cache.data, block_table, lengths, prefix_lens, alibi_slopes, out)
    refuse_gradients(q, out)
    if q.ndim != 4:
        raise ValueError("q must have shape [B, n, Hq, D]")
    batch, queries, hq, dim = q.shape
    dtype, device = q.dtype, q.device
    if dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("q must be bf16 or fp16")
    if dim != cache.head_dim:
        raise ValueError(f"the head dimension of q ({dim}) differs from the cache's ({cache.head_dim})")
    if hq == 0 or hq % cache.num_kv_heads:
        raise ValueError(f"query heads ({hq}) must be a multiple of the KV heads ({cache.num_kv_heads})")
    if not 1 <= queries <= MAX_QUERIES:
        raise ValueError(f"1 to {MAX_QUERIES} queries per request (got {queries}); longer ones belong to the prompt's "
                         "attention")
    if cache.data.device != device or block_table.device != device or lengths.device != device:
        raise ValueError("q, the cache, the block table and the lengths must be on one device")
    table = _block_table(block_table, batch)
    lengths = _per_request("lengths", lengths, batch)
    window, softcap, prefix_lens, alibi_slopes = _mask_arguments(window, softcap, prefix_lens, alibi_slopes, batch, hq,
                                                                 device)
    if not q.is_contiguous() or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != dtype or out.device != device or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError("out must be contiguous, 16-byte aligned and have the shape, type and device of q")
    elif overlaps(out, q) or overlaps(out, cache.data):
        raise ValueError("out must not overlap q or the cache")
    lse = q.new_empty((batch, queries, hq), dtype=torch.float32) if return_logsumexp else None
    width = table.shape[1]
    with device_scope(device):
        nbytes = lib().semblo_kv8_decode_workspace_bytes(batch, queries, hq, cache.num_kv_heads, dim, cache.block_size,
                                                         width, window, prefix_lens is not None)
        if nbytes < 0:
            check(int(nbytes))
        # made for this call: a recorded graph keeps its own, and calls on two streams do not share one
        workspace = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        check(lib().semblo_kv8_decode(
            q.data_ptr(), dtype_code(dtype, "decode"), batch, queries, hq, cache.num_kv_heads, dim,
            cache.data.data_ptr(), cache.scales.data_ptr(), cache.num_blocks, cache.block_size, table.data_ptr(),
            table.stride(0), width, lengths.data_ptr(), None if prefix_lens is None else prefix_lens.data_ptr(), window,
            sm_scale, softcap, None if alibi_slopes is None else alibi_slopes.data_ptr(), out.data_ptr(),
            None if lse is None else lse.data_ptr(), None if workspace is None else workspace.data_ptr(), nbytes,
            _lib.status_for(device).word.data_ptr(), raw_stream(device.index)))
    return PagedSparseAttentionResult(out, lse)
