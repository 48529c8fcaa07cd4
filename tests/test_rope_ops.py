"""Rotary tables and their scalings against the formulas, and the refusals of the rotation operators (CPU only)."""
import importlib
import math

import pytest
import torch

import __graft_entry__ as entry
from helpers import cabi, pkv_ops, pq_ops

entry.load_package()
rope_ops = importlib.import_module("mlx_metal_kernels_b200.ops.rope_ops")
layer_ops = importlib.import_module("mlx_metal_kernels_b200.ops.decode_layer_ops")
stack_mod = importlib.import_module("mlx_metal_kernels_b200.stack")
Config = rope_ops.RotaryConfig


def test_plain_frequencies_and_tables():
    cfg = Config(head_dim=128, rotary_dim=64, theta=500000.0)
    freq = rope_ops.rotary_frequencies(cfg)
    assert freq.dtype == torch.float64 and freq.shape == (32,)
    for i in (0, 1, 17, 31):
        assert float(freq[i]) == pytest.approx(500000.0 ** (-2 * i / 64), rel=1e-13)
    cos, sin = rope_ops.rotary_tables(cfg, 70000)
    assert cos.shape == sin.shape == (70000, 32) and cos.dtype == torch.float32
    # half a step of fp32 below 1, at the far end too
    for pos, i in ((69999, 0), (69999, 1), (12345, 13), (0, 0)):
        angle = pos * 500000.0 ** (-2 * i / 64)
        assert abs(float(cos[pos, i]) - math.cos(angle)) <= 2.0 ** -25 + 1e-9
        assert abs(float(sin[pos, i]) - math.sin(angle)) <= 2.0 ** -25 + 1e-9


def test_tables_near_the_stack_s_own():
    """The stack's tables (angles in fp32) agree where fp32 holds the angle: 200 positions, angle error <= 200 * 2^-23."""
    cos, sin = rope_ops.rotary_tables(Config(head_dim=128, theta=500000.0), 200)
    want = stack_mod.rope_tables(128, 500000.0, 200, "cpu")
    for a, b in zip((cos, sin), want):
        assert float((a - b).abs().max()) <= 200 * 2.0 ** -23 + 2.0 ** -23


def test_scalings():
    base = rope_ops.rotary_frequencies(Config(head_dim=64))
    linear = rope_ops.rotary_frequencies(Config(head_dim=64, scaling="linear", factor=4.0))
    assert torch.allclose(linear, base / 4, rtol=1e-14)
    ntk = rope_ops.rotary_frequencies(Config(head_dim=64, scaling="ntk", factor=4.0))
    assert float(ntk[0]) == 1.0 and float(ntk[-1]) == pytest.approx(float(base[-1]) / 4, rel=1e-12)
    cfg = Config(head_dim=128, theta=500000.0, scaling="llama3", factor=8.0, original_length=8192, low_freq_factor=1.0, high_freq_factor=4.0)
    base, got = rope_ops.rotary_frequencies(Config(head_dim=128, theta=500000.0)), rope_ops.rotary_frequencies(cfg)
    for f, g in zip(base.tolist(), got.tolist()):
        wave = 2 * math.pi / f
        if wave < 8192 / 4:
            want = f
        elif wave > 8192:
            want = f / 8
        else:
            smooth = (8192 / wave - 1) / 3
            want = (1 - smooth) * f / 8 + smooth * f
        assert g == pytest.approx(want, rel=1e-12)
    cfg = Config(head_dim=128, scaling="yarn", factor=16.0, original_length=4096)
    base, got = rope_ops.rotary_frequencies(Config(head_dim=128)), rope_ops.rotary_frequencies(cfg)
    assert float(got[0]) == float(base[0]) and float(got[-1]) == pytest.approx(float(base[-1]) / 16, rel=1e-12)
    assert bool(((got <= base) & (got >= base / 16 * (1 - 1e-12))).all())
    ratio = got / base
    assert bool((ratio[1:] <= ratio[:-1] + 1e-12).all())
    cos, _ = rope_ops.rotary_tables(cfg, 1)
    assert float(cos[0, 0]) == pytest.approx(0.1 * math.log(16.0) + 1.0, rel=2.0 ** -23)
    cos, _ = rope_ops.rotary_tables(Config(head_dim=128, scaling="yarn", factor=16.0, original_length=4096, attention_factor=1.0), 1)
    assert float(cos[0, 0]) == 1.0


@pytest.mark.parametrize("bad, match", [
    (dict(head_dim=128, rotary_dim=130), "rotary_dim"), (dict(head_dim=128, rotary_dim=3), "rotary_dim"),
    (dict(head_dim=128, rotary_dim=0), "rotary_dim"), (dict(head_dim=0), "rotary_dim"),
    (dict(head_dim=128, theta=0.0), "theta"), (dict(head_dim=128, factor=-1.0), "factor"),
    (dict(head_dim=128, scaling="dynamic"), "scaling must be one of"), (dict(head_dim=2, scaling="ntk"), "ntk"),
    (dict(head_dim=128, scaling="yarn"), "original_length"), (dict(head_dim=128, scaling="llama3"), "original_length"),
    (dict(head_dim=128, scaling="llama3", original_length=10, low_freq_factor=4.0), "low_freq_factor"),
    (dict(head_dim=128, scaling="yarn", original_length=10, beta_slow=40.0), "beta_slow"),
    (dict(head_dim=128, scaling="yarn", original_length=10, theta=1.0), "theta > 1"),
])
def test_config_refusals(bad, match):
    with pytest.raises(ValueError, match=match):
        rope_ops.rotary_frequencies(Config(**bad))


def _args(T=3, Hq=4, Hkv=2, D=32, dtype=torch.float16):
    cos, sin = rope_ops.rotary_tables(Config(head_dim=D), 16)
    return dict(q=torch.zeros(T, Hq, D, dtype=dtype), k=torch.zeros(T, Hkv, D, dtype=dtype), cos=cos, sin=sin,
                positions=torch.zeros(T, dtype=torch.int32))


@pytest.mark.parametrize("change, error, match", [
    (dict(q=torch.zeros(4, 32, dtype=torch.float16)), ValueError, "q must be"),
    (dict(k=torch.zeros(2, 2, 32, dtype=torch.float16)), ValueError, "k must be"),
    (dict(k=torch.zeros(3, 2, 64, dtype=torch.float16)), ValueError, "k must be"),
    (dict(q=torch.zeros(3, 4, 32)), TypeError, "q dtype"),
    (dict(k=torch.zeros(3, 2, 32, dtype=torch.bfloat16)), TypeError, "one dtype"),
    (dict(positions=torch.zeros(4, dtype=torch.int32)), ValueError, "positions must have shape"),
    (dict(cos=torch.zeros(16, 15)), ValueError, "cos and sin must be"),
    (dict(cos=torch.zeros(16, 17), sin=torch.zeros(16, 17)), ValueError, "cos and sin must cover"),
    (dict(cos=torch.zeros(0, 16), sin=torch.zeros(0, 16)), ValueError, "cos and sin must cover"),
    (dict(layout="split"), ValueError, "layout must be one of"),
    (dict(), cabi.B200QError, "no CPU route"),
])
def test_apply_rope_refusals(change, error, match):
    args = {**_args(), **change}
    with pytest.raises(error, match=match):
        rope_ops.apply_rope(**args)


def test_head_norm_refusals():
    a = _args()
    for weight, error, match in ((torch.zeros(31), ValueError, "norm weights must have shape"),
                                 (torch.zeros(32, dtype=torch.float64), TypeError, "norm weights must be")):
        with pytest.raises(error, match=match):
            rope_ops.head_norm_rope(a["q"], a["k"], weight, None, a["cos"], a["sin"], a["positions"])
    with pytest.raises(ValueError, match="eps"):
        rope_ops.head_norm_rope(a["q"], a["k"], None, None, a["cos"], a["sin"], a["positions"], eps=-1.0)
    with pytest.raises(cabi.ReferenceBackendUnavailable):
        rope_ops.reference_apply_rope(a["q"], a["cos"], a["sin"])


def test_in_place_refuses_shared_memory():
    check = rope_ops._check_in_place
    qkv = torch.zeros(5, 8, 32, dtype=torch.float16)
    check(qkv[:, :4], qkv[:, 4:6])                       # interleaved slices of one buffer
    check(qkv[:, 4:6], qkv[:, :4])
    check(qkv[:1, :4], qkv[:1, 4:6])
    check(torch.zeros(3, 2, 8), torch.zeros(3, 2, 8))
    for q, k in ((qkv, qkv), (qkv[:, :4], qkv[:, 3:5]), (qkv[:3], qkv[2:]), (qkv[:, 0:2], qkv[1:, 7:8].expand(-1, 1, -1)[:3, :, :].transpose(0, 1))):
        with pytest.raises(ValueError, match="in place"):
            check(q, k)
    with pytest.raises(ValueError, match="share memory"):
        check(torch.zeros(1, 4, 8).expand(3, 4, 8), None)
    with pytest.raises(ValueError, match="heads must be contiguous"):
        rope_ops._rows(torch.zeros(2, 3, 4, 8).transpose(0, 1), True)


def _cache(bits=8, pages=4, P=16, Hkv=2, D=32, G=32):
    dp = D // 2 if bits == 4 else D
    return pq_ops.PagedQuantizedKVCache(
        k_pages_q=torch.zeros(pages, P, Hkv, dp, dtype=torch.uint8), v_pages_q=torch.zeros(pages, P, Hkv, dp, dtype=torch.uint8),
        k_scales=torch.zeros(pages, P, Hkv, D // G, dtype=torch.float16), v_scales=torch.zeros(pages, P, Hkv, D // G, dtype=torch.float16),
        block_table=torch.zeros(3, 2, dtype=torch.int32), lengths=torch.zeros(3, dtype=torch.int32), bits=bits, page_size=P, group_size=G,
        original_page_shape=(pages, P, Hkv, D))


def test_append_refusals():
    cos, sin = rope_ops.rotary_tables(Config(head_dim=32), 16)
    qkv, pos = torch.zeros(3, 8 * 32, dtype=torch.float16), torch.zeros(3, dtype=torch.int32)
    call = lambda cache, qkv=qkv, pos=pos, n=4, **kw: layer_ops.norm_rope_kv_append(qkv, cos, sin, pos, cache, n, **kw)
    with pytest.raises(cabi.B200QError, match="no CPU route"):
        call(_cache())
    with pytest.raises(ValueError, match="qkv must be"):
        call(_cache(), n=5)
    with pytest.raises(TypeError, match="qkv dtype"):
        call(_cache(), qkv=qkv.float())
    with pytest.raises(ValueError, match="one token per sequence"):
        call(_cache(), qkv=qkv[:2], pos=pos[:2])
    with pytest.raises(ValueError, match="positions must have shape"):
        call(_cache(), pos=pos[:2])
    with pytest.raises(ValueError, match="sequences must have shape"):
        call(_cache(), sequences=pos[:2])
    with pytest.raises(ValueError, match="layout"):
        call(_cache(), layout="neox")
    with pytest.raises(ValueError, match="eps"):
        call(_cache(), eps=-1e-6)
    broken = _cache()
    broken.k_scales = broken.k_scales.float()
    with pytest.raises(TypeError, match="cache scales must be"):
        call(broken)
    broken = _cache()
    broken.v_pages_q = broken.v_pages_q[:, :8]
    with pytest.raises(ValueError, match="cache pages must have shape"):
        call(broken)
    broken = _cache()
    broken.k_pages_q = torch.zeros(4, 16, 32, 2, dtype=torch.uint8).transpose(2, 3)
    with pytest.raises(ValueError, match="contiguous"):
        call(broken)
    broken = _cache()
    broken.block_table = broken.block_table.long()
    with pytest.raises(TypeError, match="block_table"):
        call(broken)
    broken = _cache()
    broken.original_page_shape = None
    with pytest.raises(ValueError, match="original_page_shape"):
        call(broken)
    broken = _cache()
    broken.bits = 3
    with pytest.raises(ValueError, match="4 or 8 bits"):
        call(broken)
    pages = torch.zeros(4, 16, 2, 32, dtype=torch.bfloat16)
    table = torch.zeros(3, 2, dtype=torch.int32)
    with pytest.raises(TypeError, match="dtype of the rows"):
        pkv_ops.norm_rope_kv_append_pages(qkv, cos, sin, pos, pages, pages, table, 4)
    with pytest.raises(cabi.B200QError, match="no CPU route"):
        pkv_ops.norm_rope_kv_append_pages(qkv.bfloat16(), cos, sin, pos, pages, pages, table, 4)
    with pytest.raises(TypeError, match="positions must be int32 or int64"):
        rope_ops.int32_index(torch.zeros(3), "positions")
    assert rope_ops.int32_index(torch.tensor([5, 2 ** 40, -2 ** 40]), "positions").tolist() == [5, 2 ** 31 - 1, -1]


def test_c_abi_refuses_bad_arguments():
    """Bad sizes and null pointers come back as codes; nothing is launched (there is no GPU here)."""
    import ctypes
    lib = cabi.load()
    strides = (ctypes.c_int64 * 8)(128, 32, 128, 32, 64, 32, 64, 32)
    good = [16, 16, 16, 16, strides, None, None, 0, 0.0, 16, 16, 16, 4, 32, 0, 3, 4, 2, 32, 0, None]
    for i, v in ((0, None), (2, None), (4, None), (9, None), (11, None), (1, None), (3, None), (12, 0), (13, 0), (13, 3), (13, 34), (15, 0),
                 (16, 0), (17, -1), (18, 0), (19, 2)):
        args = list(good)
        args[i] = v
        assert lib.b200q_head_rope(*args) == -1, (i, v)
    big = list(good)
    big[18] = 2048
    assert lib.b200q_head_rope(*big) == -2
    good = [16, 256, 16, 16, 4, 32, 0, 16, None, 16, 3, 2, None, None, 0, 1e-6, 16, 8, 16, 16, 16, 16, 3, 4, 2, 32, 16, 4, 32, 0, None]
    for i, v in ((0, None), (2, None), (7, None), (9, None), (16, None), (18, None), (20, None), (1, 255), (4, 0), (5, 31), (10, 0), (10, 2),
                 (11, 0), (17, 5), (22, 0), (24, 0), (26, 0), (27, 0), (28, 0), (29, 2)):
        args = list(good)
        args[i] = v
        assert lib.b200q_norm_rope_kv_append(*args) == -1, (i, v)
