"""Rotary positions: tables (with the scalings of long contexts) and their application to query and key heads, with or
without an RMSNorm of every head in front.

The reference turns whole heads in the interleaved layout (reference_apply_rope, ops/rope_ops.py:61-75; tables
models/llama_config.py:107-124); here the layout may also be ``"half"`` (pairs ``(i, i + R/2)``), only the first ``R``
dimensions of a head may turn, and heads may be strided views of a fused projection's rows.  For the form that ends in
the cache see ``decode_layer_ops.norm_rope_kv_append`` and ``paged_kv_ops.norm_rope_kv_append_pages``.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import torch

from . import _cabi

LAYOUTS = ("interleaved", "half")
_SCALINGS = (None, "linear", "ntk", "llama3", "yarn")
_INT32_MAX = 2 ** 31 - 1
_MAX_HEAD_DIM = 1024


@dataclass(frozen=True)
class RotaryConfig:
    """Frequencies ``theta^(-2i/R)``, i < R/2, of the first ``rotary_dim`` (R; default: all) dimensions of a head, and how they
    are scaled for contexts longer than the ``original_length`` that the model was trained on:

    * ``"linear"``: every frequency divided by ``factor`` (positions interpolated);
    * ``"ntk"``: ``theta`` times ``factor^(R/(R-2))``: the lowest frequency is divided by ``factor``, the highest kept;
    * ``"llama3"``: frequencies with more than ``high_freq_factor`` turns over the original length are kept, those with fewer than
      ``low_freq_factor`` divided by ``factor``, those between blended linearly in the number of turns;
    * ``"yarn"``: the same with a blend that is linear in the dimension between ``beta_fast`` and ``beta_slow`` turns, and cos / sin
      multiplied by ``attention_factor`` (default ``0.1 ln(factor) + 1``)."""
    head_dim: int
    rotary_dim: int | None = None
    theta: float = 10000.0
    scaling: str | None = None
    factor: float = 1.0
    original_length: int | None = None
    low_freq_factor: float = 1.0
    high_freq_factor: float = 4.0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    attention_factor: float | None = None

    def validate(self) -> "RotaryConfig":
        R = self.pairs() * 2
        if self.head_dim <= 0 or R <= 0 or R > self.head_dim or (self.rotary_dim or self.head_dim) % 2:
            raise ValueError(f"rotary_dim must be even and in [2, head_dim], got {self.rotary_dim} of {self.head_dim}")
        if self.theta <= 0 or self.factor <= 0:
            raise ValueError(f"theta and factor must be positive, got {self.theta}, {self.factor}")
        if self.scaling not in _SCALINGS:
            raise ValueError(f"scaling must be one of {_SCALINGS}, got {self.scaling!r}")
        if self.scaling == "ntk" and R <= 2:
            raise ValueError("scaling 'ntk' needs rotary_dim > 2")
        if self.scaling in ("llama3", "yarn") and (self.original_length is None or self.original_length <= 0):
            raise ValueError(f"scaling {self.scaling!r} needs original_length")
        if self.scaling == "llama3" and not 0 < self.low_freq_factor < self.high_freq_factor:
            raise ValueError("low_freq_factor must be positive and below high_freq_factor")
        if self.scaling == "yarn" and not 0 < self.beta_slow < self.beta_fast:
            raise ValueError("beta_slow must be positive and below beta_fast")
        if self.scaling == "yarn" and self.theta <= 1:
            raise ValueError(f"scaling 'yarn' needs theta > 1, got {self.theta}")
        return self

    def pairs(self) -> int:
        return (self.head_dim if self.rotary_dim is None else self.rotary_dim) // 2


def rotary_frequencies(config: RotaryConfig) -> torch.Tensor:
    """Radians per position of every pair, fp64 [rotary_dim / 2] on the host."""
    config.validate()
    R = 2 * config.pairs()
    exponent = torch.arange(0, R, 2, dtype=torch.float64) / R
    theta = float(config.theta)
    if config.scaling == "ntk":
        theta *= config.factor ** (R / (R - 2))
    freq = theta ** -exponent
    if config.scaling == "linear":
        return freq / config.factor
    if config.scaling == "llama3":
        turns = config.original_length * freq / (2 * math.pi)
        keep = ((turns - config.low_freq_factor) / (config.high_freq_factor - config.low_freq_factor)).clamp(0, 1)
        return freq * (keep + (1 - keep) / config.factor)
    if config.scaling == "yarn":
        # dimension at which the original length holds `turns` turns: theta^(-2i/R) * length = 2 pi turns
        def dimension(turns):
            return R * math.log(config.original_length / (2 * math.pi * turns)) / (2 * math.log(theta))
        low = max(math.floor(dimension(config.beta_fast)), 0)
        high = min(math.ceil(dimension(config.beta_slow)), R - 1)
        ramp = ((torch.arange(R // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        return freq * (1 - ramp) + freq / config.factor * ramp
    return freq


def rotary_tables(config: RotaryConfig, length: int, device=None):
    """(cos, sin), fp32 [length, rotary_dim / 2]: angles in fp64 on the host, so that far positions keep their phase, rounded
    once.  (``stack.rope_tables`` forms the angles in fp32, as the reference does.)"""
    if length <= 0:
        raise ValueError(f"length must be positive, got {length}")
    angle = torch.arange(length, dtype=torch.float64).reshape(-1, 1) * rotary_frequencies(config).reshape(1, -1)
    gain = 1.0
    if config.scaling == "yarn":
        gain = config.attention_factor if config.attention_factor is not None else 0.1 * math.log(config.factor) + 1.0
    return tuple((t * gain).to(torch.float32).contiguous().to(device) for t in (torch.cos(angle), torch.sin(angle)))


# ---------------------------------------------------------------------------------------------
# shared checks
# ---------------------------------------------------------------------------------------------
def layout_code(layout: str) -> int:
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {LAYOUTS}, got {layout!r}")
    return LAYOUTS.index(layout)


def check_tables(cos, sin, head_dim: int):
    """cos / sin as the kernels read them: fp32 contiguous [table_len, rotary_dim / 2]."""
    if cos.ndim != 2 or cos.shape != sin.shape:
        raise ValueError(f"cos and sin must be [table_len, rotary_dim/2] of one shape, got {tuple(cos.shape)}, {tuple(sin.shape)}")
    if cos.shape[0] == 0 or cos.shape[1] == 0 or 2 * cos.shape[1] > head_dim:
        raise ValueError(f"cos and sin must cover between one pair and the {head_dim} dimensions of a head, got {tuple(cos.shape)}")
    return _cabi.contiguous(cos.to(torch.float32)), _cabi.contiguous(sin.to(torch.float32))


def int32_index(t, what: str):
    """Integer indices as contiguous int32; values that int32 does not hold become its ends, which no table reaches."""
    if t.dtype == torch.int32:
        return _cabi.contiguous(t)
    if t.dtype != torch.int64:
        raise TypeError(f"{what} must be int32 or int64, got {t.dtype}")
    return _cabi.contiguous(t.clamp(-1, _INT32_MAX).to(torch.int32))


def check_head_weights(weights, head_dim: int):
    """Per-head norm weights [head_dim] (or None) in one dtype the kernels read."""
    given = [w for w in weights if w is not None]
    for w in given:
        if tuple(w.shape) != (head_dim,):
            raise ValueError(f"norm weights must have shape {(head_dim,)}, got {tuple(w.shape)}")
        if w.dtype not in (torch.float16, torch.bfloat16, torch.float32):
            raise TypeError(f"norm weights must be float16, bfloat16 or float32, got {w.dtype}")
    if len({w.dtype for w in given}) > 1:
        weights = [None if w is None else w.to(torch.float32) for w in weights]
    return [_cabi.contiguous(w) for w in weights], (_cabi.dtype_code(given[0].dtype) if len({w.dtype for w in given}) == 1 else _cabi.F32)


def _rows(x, inplace: bool):
    """x [..., H, D] as [T, H, D] with contiguous heads, without a copy where the strides allow it."""
    T = math.prod(x.shape[:-2])
    if x.stride(-1) == 1 or x.shape[-1] == 1:
        try:
            return x.view(T, *x.shape[-2:])
        except RuntimeError:
            pass
    if inplace:
        raise ValueError("in place, heads must be contiguous and the leading dimensions of one stride")
    return x.contiguous().view(T, *x.shape[-2:])


def _span(x):
    """Elements between the first and one past the last of a view, and whether no two of its elements share memory."""
    dims = sorted((st, n) for n, st in zip(x.shape, x.stride()) if n > 1)
    reach = 1
    for st, n in dims:
        if st < reach:
            return reach, False
        reach = st * (n - 1) + reach
    return reach, True


def _check_in_place(q, k):
    for x in (q, k):
        if x is not None and not _span(x)[1]:
            raise ValueError("in place, no two elements of q or k may share memory")
    if k is None:
        return
    size = q.element_size()
    first, second = sorted(((x.data_ptr() // size, _span(x)[0], x) for x in (q, k)), key=lambda e: e[0])
    if first[0] + first[1] <= second[0]:
        return
    # interleaved slices of one buffer: the rows of one must fall between the rows of the other
    step = first[2].stride(0)
    apart = second[0] - first[0]
    row = [_span(e[2][0])[0] for e in (first, second)]
    one_row = first[2].shape[0] == 1 and second[2].shape[0] == 1
    if one_row or second[2].stride(0) != step or apart < row[0] or apart + row[1] > step:
        raise ValueError("in place, q and k must not overlap")


def _head_rope(q, k, weights, cos, sin, positions, eps, layout, inplace, who):
    if q.ndim < 3:
        raise ValueError(f"q must be [..., heads, head_dim] with at least one leading dimension, got {tuple(q.shape)}")
    lead, D = tuple(q.shape[:-2]), q.shape[-1]
    if k is not None and (k.ndim != q.ndim or tuple(k.shape[:-2]) != lead or k.shape[-1] != D):
        raise ValueError(f"k must be [..., heads, head_dim] beside q {tuple(q.shape)}, got {tuple(k.shape)}")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"q dtype must be float16 or bfloat16, got {q.dtype}")
    if k is not None and k.dtype != q.dtype:
        raise TypeError(f"q and k must have one dtype, got {q.dtype}, {k.dtype}")
    if tuple(positions.shape) != lead and not (len(lead) == 2 and tuple(positions.shape) == lead[1:]):
        raise ValueError(f"positions must have shape {lead}{' or ' + str(lead[1:]) if len(lead) == 2 else ''}, got {tuple(positions.shape)}")
    if not 0 < D <= _MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be in [1, {_MAX_HEAD_DIM}], got {D}")
    half = layout_code(layout)
    cos, sin = check_tables(cos, sin, D)
    weights, w_dtype = check_head_weights(weights, D)
    device = _cabi.require_cuda(q, k, cos, sin, positions, *weights)
    positions = int32_index(positions.expand(lead), "positions")
    q3, k3 = _rows(q, inplace), None if k is None else _rows(k, inplace)
    if inplace:
        _check_in_place(q3, k3)
        q_out, k_out = q, k
        qo3, ko3 = q3, k3
    else:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=device)
        k_out = None if k is None else torch.empty(k.shape, dtype=k.dtype, device=device)
        qo3, ko3 = q_out.view(q3.shape), None if k is None else k_out.view(k3.shape)
    T, Hq = q3.shape[:2]
    if T == 0 or (Hq == 0 and (k is None or k3.shape[1] == 0)):
        return q_out, k_out
    if Hq == 0:
        raise ValueError("q must have at least one head")
    if k3 is not None and k3.shape[1] == 0:
        k3 = None
    strides = [q3.stride(0), q3.stride(1), qo3.stride(0), qo3.stride(1)]
    strides += [0] * 4 if k3 is None else [k3.stride(0), k3.stride(1), ko3.stride(0), ko3.stride(1)]
    with _cabi.on_device(device):
        _cabi.check(
            _cabi.load().b200q_head_rope(q3.data_ptr(), _cabi.ptr(k3), qo3.data_ptr(), None if k3 is None else ko3.data_ptr(),
                                         (ctypes.c_int64 * 8)(*strides), _cabi.ptr(weights[0]), _cabi.ptr(weights[1]), w_dtype,
                                         float(eps), cos.data_ptr(), sin.data_ptr(), positions.data_ptr(), cos.shape[0],
                                         2 * cos.shape[1], half, T, Hq, 0 if k3 is None else k3.shape[1], D,
                                         _cabi.dtype_code(q.dtype), _cabi.stream()),
            who)
    return q_out, k_out


def reference_apply_rope(x, cos, sin):
    _cabi.reference_unavailable("reference_apply_rope")


def apply_rope(q, k, cos, sin, positions, *, layout: str = "interleaved", inplace: bool = False):
    """Turns the heads of q [..., Hq, D] and k [..., Hkv, D] (or None), fp16 / bf16, by ``positions`` [...] (or [S] for [B, S]
    leading dimensions).  ``cos`` / ``sin`` [table_len, R/2] as ``rotary_tables`` builds them; the first R dimensions of a head
    turn.  fp32, rounded once.  Returns (q, k): new contiguous tensors, or the arguments themselves with ``inplace``.

    q and k may be strided views (slices of the fused rows).  A position outside the table leaves its heads unturned and is
    reported by ``_cabi.device_status()`` (event 6); nothing is read on the host, so the call can be captured."""
    if not inplace:
        out = _cabi.host().head_rope(q, k, None, None, cos, sin, positions, 0.0, layout)
        if out is not None:
            return out
    return _head_rope(q, k, (None, None), cos, sin, positions, 0.0, layout, inplace, "apply_rope")


def head_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, *, eps: float = 1e-6, layout: str = "interleaved",
                   inplace: bool = False):
    """``apply_rope`` with an RMSNorm of every head in front, in the same pass: y = x * rsqrt(mean(x^2) + eps) * weight over the
    whole head, not rounded before the rotation.  A weight [D] of None leaves its heads as they are."""
    if not inplace:
        out = _cabi.host().head_rope(q, k, q_weight, k_weight, cos, sin, positions, eps, layout)
        if out is not None:
            return out
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    return _head_rope(q, k, (q_weight, k_weight), cos, sin, positions, eps, layout, inplace, "head_norm_rope")


def append_launch(qkv, cos, sin, positions, sequences, block_table, n_heads, weights, eps, layout, kv_bits, k_pages, v_pages, k_scales,
                  v_scales, page_shape, group_size, who):
    """Checks and launch of the append form for both kinds of pages; ``page_shape`` (NUM_PAGES, PAGE_SIZE, Hkv, D)."""
    num_pages, page_size, Hkv, D = page_shape
    if qkv.ndim != 2 or qkv.shape[1] != (n_heads + 2 * Hkv) * D or n_heads <= 0:
        raise ValueError(f"qkv must be [T, (n_heads + 2 * {Hkv}) * {D}] with n_heads = {n_heads}, got {tuple(qkv.shape)}")
    if qkv.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"qkv dtype must be float16 or bfloat16, got {qkv.dtype}")
    T = qkv.shape[0]
    if block_table.ndim != 2 or block_table.dtype != torch.int32 or not block_table.is_contiguous():
        raise TypeError("block_table must be a contiguous int32 tensor [B, MAX_BLOCKS]")
    B, max_blocks = block_table.shape
    if tuple(positions.shape) != (T,):
        raise ValueError(f"positions must have shape {(T,)}, got {tuple(positions.shape)}")
    if sequences is None:
        if T != B:
            raise ValueError(f"without sequences there must be one token per sequence: {T} tokens, {B} sequences")
    elif tuple(sequences.shape) != (T,):
        raise ValueError(f"sequences must have shape {(T,)}, got {tuple(sequences.shape)}")
    if not 0 < D <= _MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be in [1, {_MAX_HEAD_DIM}], got {D}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    half = layout_code(layout)
    cos, sin = check_tables(cos, sin, D)
    weights, w_dtype = check_head_weights(weights, D)
    for t in (k_pages, v_pages, k_scales, v_scales):
        if t is not None and not t.is_contiguous():
            raise ValueError("pages and scales are written in place: they must be contiguous")
    device = _cabi.require_cuda(qkv, cos, sin, positions, sequences, block_table, k_pages, v_pages, k_scales, v_scales, *weights)
    q_out = torch.empty((T, n_heads, D), dtype=qkv.dtype, device=device)
    if T == 0:
        return q_out
    if qkv.stride(1) != 1 or qkv.stride(0) < qkv.shape[1]:
        qkv = qkv.contiguous()
    positions = int32_index(positions, "positions")
    sequences = None if sequences is None else int32_index(sequences, "sequences")
    with _cabi.on_device(device):
        _cabi.check(
            _cabi.load().b200q_norm_rope_kv_append(qkv.data_ptr(), qkv.stride(0), cos.data_ptr(), sin.data_ptr(), cos.shape[0],
                                                   2 * cos.shape[1], half, positions.data_ptr(), _cabi.ptr(sequences),
                                                   block_table.data_ptr(), B, max_blocks, _cabi.ptr(weights[0]), _cabi.ptr(weights[1]),
                                                   w_dtype, float(eps), q_out.data_ptr(), kv_bits, k_pages.data_ptr(), v_pages.data_ptr(),
                                                   _cabi.ptr(k_scales), _cabi.ptr(v_scales), T, n_heads, Hkv, D, page_size, num_pages,
                                                   group_size, _cabi.dtype_code(qkv.dtype), _cabi.stream()),
            who)
    return q_out
