"""Refusals of the adapter operators (CPU only)."""
import importlib

import pytest
import torch

import __graft_entry__ as entry
from helpers import cabi, random_quant_case

entry.load_package()
lora = importlib.import_module("mlx_metal_kernels_b200.ops.lora_ops")


def case(rows=2, N=32, K=64, L=3, R=4, dtype=torch.float16):
    w, s, z = random_quant_case(4, N, K, 32, 1)
    return dict(x=torch.zeros(rows, K, dtype=dtype), w=w, scales=s, zeros=z,
                adapters=lora.LoraAdapters(torch.zeros(L, R, K, dtype=dtype), torch.zeros(L, N, R, dtype=dtype)),
                adapter_ids=torch.zeros(rows, dtype=torch.int32))


@pytest.mark.parametrize("change, error, match", [
    (dict(), cabi.B200QError, "no CPU route"),
    (dict(x=torch.zeros(2, 64)), TypeError, "x dtype"),
    (dict(x=torch.zeros(2, 64, dtype=torch.bfloat16)), TypeError, "dtype of the rows"),
    (dict(x=torch.zeros(64, dtype=torch.float16)), ValueError, "x must have shape"),
    (dict(adapter_ids=torch.zeros(3, dtype=torch.int32)), ValueError, "adapter_ids must have shape"),
    (dict(adapter_ids=torch.zeros(2)), TypeError, "adapter_ids must be"),
    (dict(residual=torch.zeros(2, 31, dtype=torch.float16)), ValueError, "residual must have shape"),
    (dict(bits=8), ValueError, "q8 weights"),
    (dict(group_size=0), ValueError, "group_size"),
    (dict(backend="vulkan"), ValueError, "backend must be one of"),
    (dict(backend="reference"), cabi.ReferenceBackendUnavailable, "not part of this library"),
    (dict(adapters=lora.LoraAdapters(torch.zeros(3, 4, 32, dtype=torch.float16), torch.zeros(3, 32, 4, dtype=torch.float16))), ValueError, "do not fit"),
    (dict(adapters=lora.LoraAdapters(torch.zeros(3, 4, 64, dtype=torch.float16), torch.zeros(3, 31, 4, dtype=torch.float16))), ValueError, "do not fit"),
])
def test_refusals(change, error, match):
    args = {**case(), **change}
    with pytest.raises(error, match=match):
        lora.lora_quantized_linear(**args)


@pytest.mark.parametrize("a, b, more, error, match", [
    ((3, 4, 64), (3, 32, 5), {}, ValueError, r"a must be \[L,R,K\]"), ((2, 4, 64), (3, 32, 4), {}, ValueError, r"a must be \[L,R,K\]"),
    ((4, 64), (32, 4), {}, ValueError, r"a must be \[L,R,K\]"), ((0, 4, 64), (0, 32, 4), {}, ValueError, r"a must be \[L,R,K\]"),
    ((3, 4, 64), (3, 32, 4), dict(scaling=torch.zeros(3, dtype=torch.float16)), ValueError, "scaling must be"),
    ((3, 4, 64), (3, 32, 4), dict(scaling=torch.zeros(2)), ValueError, "scaling must be"),
    ((3, 4, 64), (3, 32, 4), dict(ranks=torch.zeros(3)), ValueError, "ranks must be"),
])
def test_adapter_refusals(a, b, more, error, match):
    with pytest.raises(error, match=match):
        lora.LoraAdapters(torch.zeros(a, dtype=torch.float16), torch.zeros(b, dtype=torch.float16), **more).validate()


def test_adapter_dtypes_and_rows():
    with pytest.raises(TypeError, match="one dtype"):
        lora.LoraAdapters(torch.zeros(1, 2, 8), torch.zeros(1, 8, 2)).validate()
    with pytest.raises(TypeError, match="one dtype"):
        lora.LoraAdapters(torch.zeros(1, 2, 8, dtype=torch.float16), torch.zeros(1, 8, 2, dtype=torch.bfloat16)).validate()
    c = case()
    with pytest.raises(ValueError, match="y must be"):
        lora.lora_add(torch.zeros(3, 32, dtype=torch.float16), c["x"], c["adapters"], c["adapter_ids"])
    with pytest.raises(ValueError, match="y must be"):
        lora.lora_add(torch.zeros(2, 32), c["x"], c["adapters"], c["adapter_ids"])
    with pytest.raises(cabi.B200QError, match="no CPU route"):
        lora.lora_add(torch.zeros(2, 32, dtype=torch.float16), c["x"], c["adapters"], c["adapter_ids"])


def test_safe_mode_is_refused(monkeypatch):
    monkeypatch.setenv("MLX_METAL_CI_SAFE_MODE", "1")
    with pytest.raises(cabi.ReferenceBackendUnavailable):
        lora.lora_quantized_linear(**case())


def test_c_abi_refuses_bad_arguments():
    lib = cabi.load()
    good = [16, 16, 16, 16, 16, None, None, 16, 2, 32, 64, 3, 4, 0, 16, 1 << 20, None]
    for i, v in ((0, None), (2, None), (3, None), (4, None), (7, None), (8, 0), (9, 0), (10, 0), (11, 0), (12, 0), (13, 2)):
        args = list(good)
        args[i] = v
        assert lib.b200q_lora_add(*args) == -1, (i, v)
    for i, v in ((14, None), (15, 31)):
        args = list(good)
        args[i] = v
        assert lib.b200q_lora_add(*args) == -4, (i, v)
    assert lib.b200q_lora_workspace_bytes(2, 4) == 32 and lib.b200q_lora_workspace_bytes(0, 4) == 0
    good = [4, 16, 16, 16, 16, None, 16, 16, 16, None, None, 16, 2, 32, 64, 32, 3, 4, 0, 0, 16, 1 << 20, None]
    for i, v in ((0, 5), (1, None), (2, None), (3, None), (6, None), (7, None), (8, None), (11, None), (12, 0), (13, 0), (14, 0), (15, 0), (16, 0),
                 (17, 0), (18, 2), (19, 3)):
        args = list(good)
        args[i] = v
        assert lib.b200q_lora_qmatvec(*args) == -1, (i, v)
    for i, v in ((20, None), (21, 2 * 32 * 4)):
        args = list(good)
        args[i] = v
        assert lib.b200q_lora_qmatvec(*args) == -4, (i, v)
    for i in (13, 14):
        args = list(good)
        args[i] = 2 ** 31
        assert lib.b200q_lora_qmatvec(*args) == -2
    assert lib.b200q_lora_qmatvec_workspace_bytes(2, 32, 4) >= 2 * 32 * 4 + 32 and lib.b200q_lora_qmatvec_workspace_bytes(0, 32, 4) == 0


def test_c_abi_refuses_workspaces_that_are_not_aligned():
    lib = cabi.load()
    assert lib.b200q_lora_add(16, 16, 16, 16, 16, None, None, 16, 2, 32, 64, 3, 4, 0, 8, 1 << 20, None) == -4
    assert lib.b200q_lora_qmatvec(4, 16, 16, 16, 16, None, 16, 16, 16, None, None, 16, 2, 32, 64, 32, 3, 4, 0, 0, 24, 1 << 20, None) == -4
