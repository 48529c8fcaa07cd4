"""Low-rank adapters of many requests beside a shared quantized projection.

A decode batch (or a chunk of prompts) goes through one set of quantized weights; every row may add the correction of its own adapter:
``y[t] = W x[t] + scaling[l] * B[l] (A[l] x[t])`` with ``l = adapter_ids[t]``, or nothing where the id is negative.  The reference has no
adapters; the shared part is its ``quantized_linear`` (ops/mlp_block_ops.py:77-101).
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Any

import torch

from . import _cabi
from .mlp_block_ops import _normalize_hidden_input, _restore_hidden_output, _validate_quantized_linear_shapes
from .quant_ops import _resolve_matvec_backend
from .rope_ops import int32_index


@dataclass
class LoraAdapters:
    """Factors of ``L`` adapters of one projection: ``a`` [L, R, K] and ``b`` [L, N, R] in the dtype of the rows (fp16 / bf16), ``scaling``
    fp32 [L] (None: 1) and ``ranks`` int32 [L] (None: R): adapter l uses the first ``ranks[l]`` rows of ``a[l]`` and columns of ``b[l]``."""
    a: Any
    b: Any
    scaling: Any = None
    ranks: Any = None

    def validate(self) -> "LoraAdapters":
        a, b = self.a, self.b
        if a.ndim != 3 or b.ndim != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2] or 0 in a.shape or 0 in b.shape:
            raise ValueError(f"a must be [L,R,K] and b [L,N,R], got {tuple(a.shape)}, {tuple(b.shape)}")
        if a.dtype not in (torch.float16, torch.bfloat16) or b.dtype != a.dtype:
            raise TypeError(f"a and b must be float16 or bfloat16 of one dtype, got {a.dtype}, {b.dtype}")
        for name, t, dtype in (("scaling", self.scaling, torch.float32), ("ranks", self.ranks, torch.int32)):
            if t is not None and (tuple(t.shape) != (a.shape[0],) or t.dtype != dtype):
                raise ValueError(f"{name} must be {dtype} of shape {(a.shape[0],)}, got {t.dtype} {tuple(t.shape)}")
        return self


def _check(x2d, adapters, adapter_ids, lead, out_dim):
    """(adapter ids as the kernels read them, int32 [rows])"""
    adapters.validate()
    if x2d.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"x dtype must be float16 or bfloat16, got {x2d.dtype}")
    if adapters.a.dtype != x2d.dtype:
        raise TypeError(f"adapters must have the dtype of the rows, got {adapters.a.dtype} and {x2d.dtype}")
    if adapters.a.shape[2] != x2d.shape[1] or adapters.b.shape[1] != out_dim:
        raise ValueError(f"adapters of [K,N] = {(adapters.a.shape[2], adapters.b.shape[1])} do not fit rows of {x2d.shape[1]} -> {out_dim}")
    shape = tuple(adapter_ids.shape)
    if shape != lead and not (len(lead) == 2 and shape == lead[:1]):
        raise ValueError(f"adapter_ids must have shape {lead}{' or ' + str(lead[:1]) if len(lead) == 2 else ''}, got {shape}")
    if shape != lead:
        adapter_ids = adapter_ids.reshape(-1, 1).expand(lead)
    return int32_index(adapter_ids.reshape(math.prod(lead)), "adapter_ids")


def _factors(adapters):
    """(tensors the kernels read - to be kept until the launch -, their addresses and sizes as the C calls take them)"""
    a, b = _cabi.contiguous(adapters.a), _cabi.contiguous(adapters.b)
    scaling, ranks = _cabi.contiguous(adapters.scaling), _cabi.contiguous(adapters.ranks)
    return (a, b, scaling, ranks), (a.data_ptr(), b.data_ptr(), _cabi.ptr(scaling), _cabi.ptr(ranks)), (a.shape[0], a.shape[1])


def _workspace(nbytes, device):
    return torch.empty(max(16, nbytes), dtype=torch.uint8, device=device)


def lora_add(y, x, adapters: LoraAdapters, adapter_ids):
    """y + scaling * B (A x) with the adapter of every row: rows x [B,K] / [B,S,K] and what the shared projection made of them, y [B,N] /
    [B,S,N]; ``adapter_ids`` [B] / [B,S] (or [B] for [B,S] rows: one per sequence), int32 or int64, negative: none.  fp32, rounded once.
    An id beyond the stack counts as none and is reported by ``_cabi.device_status()`` (event 10)."""
    x2d, shape = _normalize_hidden_input(x)
    if tuple(y.shape[:-1]) != shape[:-1] or y.dtype != x.dtype:
        raise ValueError(f"y must be {shape[:-1]} rows in {x.dtype}, got {tuple(y.shape)} {y.dtype}")
    ids = _check(x2d, adapters, adapter_ids, shape[:-1], y.shape[-1])
    device = _cabi.require_cuda(x2d, y, adapters.a, adapters.b, adapters.scaling, adapters.ranks, ids)
    out = torch.empty(y.shape, dtype=y.dtype, device=device)
    if out.numel() == 0:
        return out
    with _cabi.on_device(device):
        x2d, y = _cabi.contiguous(x2d), _cabi.contiguous(y)
        rows, K = x2d.shape
        keep, factors, (L, R) = _factors(adapters)
        lib = _cabi.load()
        ws = _workspace(lib.b200q_lora_workspace_bytes(rows, R), device)
        _cabi.check(lib.b200q_lora_add(x2d.data_ptr(), y.data_ptr(), out.data_ptr(), *factors, ids.data_ptr(), rows, y.shape[-1], K, L, R,
                                       _cabi.dtype_code(x.dtype), ws.data_ptr(), ws.numel(), _cabi.stream()), "b200q_lora_add")
    return out


def lora_quantized_linear(x, w, scales, zeros, adapters: LoraAdapters, adapter_ids, *, bits=4, group_size=32, residual=None, backend="auto"):
    """``quantized_linear`` with the adapter of every row: [B,K] / [B,S,K] -> N features, y = W x + scaling * B (A x), plus ``residual``
    [.., N] where given.  All sums are fp32 and rounded once, at the end."""
    out = _cabi.host().lora_linear(bits, x, w, scales, zeros, group_size, backend, adapters, adapter_ids, residual)
    if out is not None:
        return out
    x2d, shape = _normalize_hidden_input(x)
    _, out_dim = _validate_quantized_linear_shapes(x2d, w, scales, zeros, bits=bits, group_size=group_size, name="lora_quantized_linear")
    _resolve_matvec_backend(backend, "lora_quantized_linear")
    ids = _check(x2d, adapters, adapter_ids, shape[:-1], out_dim)
    if residual is not None and tuple(residual.shape) != (*shape[:-1], out_dim):
        raise ValueError(f"residual must have shape {(*shape[:-1], out_dim)}, got {tuple(residual.shape)}")
    device = _cabi.require_cuda(x2d, w, scales, zeros, residual, adapters.a, adapters.b, adapters.scaling, adapters.ranks, ids)
    if x2d.shape[0] == 0:
        return torch.empty((*shape[:-1], out_dim), dtype=x.dtype, device=device)
    with _cabi.on_device(device):
        x2d, w = _cabi.contiguous(x2d), _cabi.contiguous(w.to(torch.uint8))
        scales, zeros = _cabi.scale_pair(scales, zeros)
        residual = None if residual is None else _cabi.contiguous(residual.reshape(-1, out_dim).to(x.dtype))
        rows, K = x2d.shape
        keep, factors, (L, R) = _factors(adapters)
        y = torch.empty((rows, out_dim), dtype=x.dtype, device=device)
        ws = _workspace(_cabi.load().b200q_lora_qmatvec_workspace_bytes(rows, out_dim, R), device)
        _cabi.call_with_scratch("b200q_lora_qmatvec", rows, K, x2d, bits, x2d.data_ptr(), w.data_ptr(), scales.data_ptr(), _cabi.ptr(zeros),
                                _cabi.ptr(residual), y.data_ptr(), *factors, ids.data_ptr(), rows, out_dim, K, group_size, L, R,
                                _cabi.dtype_code(x.dtype), _cabi.dtype_code(scales.dtype), ws.data_ptr(), ws.numel(), _cabi.stream())
    return _restore_hidden_output(y, shape)
