"""Rotary positions for the queries and keys of a layer: q_post / k_post from q_pre / k_pre.

The sparse path routes with the vectors before the rotation and attends with the ones after it, so a
layer keeps both; :func:`apply_rotary` makes the second from the first in one launch.  Half and
interleaved layouts, a rotated part of the head, and frequencies scaled for contexts longer than the
model was trained on (:func:`rotary_frequencies`).  The reference leaves this step to the engine's
rotary layer (semblo/vllm_plugin/model.py:1130-1167 receives both tensors)."""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from ._lib import check, device_scope, dtype_code, lib, overlaps, raw_stream, refuse_gradients, require_cuda

_SCALING_KEYS = {"linear": {"factor"}, "ntk": {"factor"},
                 "yarn": {"factor", "original_max_position", "beta_fast", "beta_slow", "attention_factor"},
                 "wavelength": {"factor", "original_max_position", "low_freq_factor", "high_freq_factor"}}
_SCALING_REQUIRED = {"linear": {"factor"}, "ntk": {"factor"}, "yarn": {"factor", "original_max_position"},
                     "wavelength": _SCALING_KEYS["wavelength"]}


@dataclass(frozen=True)
class RotaryFrequencies:
    """What a layer's rotation needs besides the positions."""

    inv_freq: torch.Tensor            # [R / 2] float64: angle per position of each pair
    attention_scale: float = 1.0      # on cos and sin

    def __post_init__(self) -> None:
        if self.inv_freq.ndim != 1 or self.inv_freq.dtype != torch.float64 or not self.inv_freq.is_contiguous():
            raise ValueError("inv_freq must be a contiguous float64 vector (angles of far positions need 64 bits)")

    @property
    def rotary_dim(self) -> int:
        return 2 * int(self.inv_freq.shape[0])


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, *, scaling: dict | None = None,
                       device="cuda") -> RotaryFrequencies:
    """Frequencies base^(-2i / rotary_dim), scaled as ``scaling`` says:

    ``{"type": "linear", "factor": s}``       positions are divided by s;
    ``{"type": "ntk", "factor": s}``          the base grows by s^(R / (R - 2)): the lowest frequency is divided
                                              by s, the highest stays;
    ``{"type": "yarn", "factor": s, "original_max_position": L, "beta_fast": 32, "beta_slow": 1,
    "attention_factor": 0.1 ln s + 1}``       pairs that turn more than beta_fast times within L stay, those below
                                              beta_slow are divided by s, a linear ramp over the pairs between;
    ``{"type": "wavelength", "factor": s, "original_max_position": L, "low_freq_factor": a,
    "high_freq_factor": b}``                  the same with the ramp linear in the turns, between a and b."""
    r = int(rotary_dim)
    if r <= 0 or r % 2:
        raise ValueError(f"rotary_dim must be positive and even (got {rotary_dim})")
    base = float(base)
    if not base > 1.0:
        raise ValueError(f"the rotary base must be above 1 (got {base})")
    spec = dict(scaling or {})
    kind = spec.pop("type", None)
    if scaling and kind not in _SCALING_KEYS:
        raise ValueError(f"unknown rotary scaling {kind!r} (known: {sorted(_SCALING_KEYS)})")
    if kind is not None:
        extra, missing = set(spec) - _SCALING_KEYS[kind], _SCALING_REQUIRED[kind] - set(spec)
        if extra or missing:
            raise ValueError(f"rotary scaling {kind!r}: unknown keys {sorted(extra)}, missing keys {sorted(missing)}")
    factor = float(spec.get("factor", 1.0))
    if not factor >= 1.0:
        raise ValueError(f"the rotary scaling factor must be at least 1 (got {factor})")
    length = float(spec.get("original_max_position", 1.0))
    if not length >= 1.0:
        raise ValueError(f"original_max_position must be at least 1 (got {length})")
    pairs = torch.arange(r // 2, dtype=torch.float64)
    scale = 1.0
    if kind == "ntk":
        base *= factor ** (r / max(r - 2, 1))
    inv = base ** (-2.0 * pairs / r)
    if kind == "linear":
        inv = inv / factor
    elif kind == "yarn":
        def pair_at(turns: float) -> float:          # the (fractional) pair that turns this often within length
            return r * math.log(length / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
        fast, slow = float(spec.get("beta_fast", 32.0)), float(spec.get("beta_slow", 1.0))
        if not 0 < slow <= fast:
            raise ValueError(f"rotary scaling 'yarn': 0 < beta_slow <= beta_fast is required (got {slow}, {fast})")
        lo, hi = max(math.floor(pair_at(fast)), 0), min(math.ceil(pair_at(slow)), r - 1)
        ramp = ((pairs - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
        inv = inv * (1.0 - ramp) + inv / factor * ramp
        scale = float(spec.get("attention_factor", 0.1 * math.log(factor) + 1.0))
    elif kind == "wavelength":
        a, b = float(spec["low_freq_factor"]), float(spec["high_freq_factor"])
        if not 0 < a < b:
            raise ValueError(f"rotary scaling 'wavelength': 0 < low_freq_factor < high_freq_factor (got {a}, {b})")
        keep = ((length * inv / (2.0 * math.pi) - a) / (b - a)).clamp(0.0, 1.0)
        inv = inv * (keep + (1.0 - keep) / factor)
    return RotaryFrequencies(inv.to(device), scale)


def _check_rows(name: str, x: torch.Tensor, tokens: int, dim: int, dtype, device) -> tuple:
    """The strides of x [tokens, heads, dim]."""
    shape, strides = x.shape, x.stride()
    if len(shape) != 3 or shape[0] != tokens or shape[2] != dim:
        raise ValueError(f"{name} must have shape [{tokens}, heads, {dim}] (got {tuple(shape)})")
    if strides[2] != 1 and dim > 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")
    if x.dtype != dtype:
        raise ValueError("q_pre, k_pre and the outputs must have one dtype")
    if x.device != device:
        raise ValueError(f"the tensors of a call must be on one device ({name} is on {x.device}, q_pre on {device})")
    return strides


def _check_output(name: str, y: torch.Tensor, x: torch.Tensor) -> tuple:
    strides = _check_rows(name, y, x.shape[0], x.shape[2], x.dtype, x.device)
    if y.shape != x.shape:
        raise ValueError(f"{name} must have the shape of its input")
    if any(n > 1 and s == 0 for n, s in zip(y.shape, strides)):
        raise ValueError(f"{name} must not repeat memory")
    if (x.data_ptr() != y.data_ptr() or x.stride() != strides) and overlaps(x, y):
        raise ValueError(f"{name} overlaps its input without being it")
    return strides


def apply_rotary(q_pre: torch.Tensor, k_pre: torch.Tensor | None, positions: torch.Tensor,
                 frequencies: RotaryFrequencies, *, interleaved: bool = False, inverse: bool = False,
                 q_out: torch.Tensor | None = None,
                 k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Rotate ``q_pre`` [T, Hq, D] and ``k_pre`` [T, Hkv, D] (or None) by their ``positions`` [T].

    bf16, fp16 or fp32, any token and head strides (views of a fused projection); int32 or int64 positions.
    The first ``frequencies.rotary_dim`` dimensions are rotated: pair i is (x_i, x_{i + R/2}), or (x_2i, x_2i+1)
    with ``interleaved``; the others are copied.  ``inverse`` rotates back (the transpose).  ``q_out`` / ``k_out``
    receive the result; either may be its input itself (in place), and must not share an element with the other
    input or output (slices of one fused buffer do not; the C entry looks at strides).  Angles are formed in 64 bits."""
    require_cuda(q_pre, k_pre, positions, q_out, k_out)
    refuse_gradients(q_pre, k_pre, q_out, k_out)
    if q_pre.ndim != 3:
        raise ValueError("q_pre must have shape [T, Hq, D]")
    tokens, hq, dim = q_pre.shape
    dtype, device = q_pre.dtype, q_pre.device
    code = dtype_code(dtype, "rotary")
    qs = _check_rows("q_pre", q_pre, tokens, dim, dtype, device)
    if positions.ndim != 1 or positions.shape[0] != tokens or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be one int32 or int64 per token")
    inv_freq = frequencies.inv_freq
    rotary_dim = 2 * inv_freq.shape[0]
    if rotary_dim > dim:
        raise ValueError(f"rotary_dim {rotary_dim} exceeds the head dimension {dim}")
    if positions.device != device or inv_freq.device != device:
        raise ValueError(f"the positions ({positions.device}) and frequencies ({inv_freq.device}) must be on the "
                         f"device of q_pre ({device})")
    if q_out is None:
        q_out, qos = torch.empty_like(q_pre, memory_format=torch.contiguous_format), (hq * dim, dim)
    else:
        qos = _check_output("q_out", q_out, q_pre)
    hkv, k_args = 0, (None, 0, 0, None, 0, 0, 0)
    if k_pre is None:
        if k_out is not None:
            raise ValueError("k_out is given without k_pre")
    else:
        ks = _check_rows("k_pre", k_pre, tokens, dim, dtype, device)
        hkv = k_pre.shape[1]
        if k_out is None:
            k_out, kos = torch.empty_like(k_pre, memory_format=torch.contiguous_format), (hkv * dim, dim)
        else:
            kos = _check_output("k_out", k_out, k_pre)
        if hkv:
            k_args = (k_pre.data_ptr(), ks[0], ks[1], k_out.data_ptr(), kos[0], kos[1], hkv)
    if not positions.is_contiguous():
        positions = positions.contiguous()
    with device_scope(device):
        check(lib().semblo_rotary(
            q_pre.data_ptr(), qs[0], qs[1], q_out.data_ptr(), qos[0], qos[1], hq,
            *k_args, tokens, dim, rotary_dim, code, positions.data_ptr(), positions.dtype == torch.int64,
            inv_freq.data_ptr(), frequencies.attention_scale, interleaved, inverse, raw_stream(device.index)))
    return q_out, k_out
