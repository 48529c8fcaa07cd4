"""GPU rotation, head norms and appends against the formulas in 64 bits."""
import importlib

import pytest
import torch

import __graft_entry__ as entry
from helpers import cabi, gen, pkv_ops, pq_ops, synth

pytestmark = pytest.mark.gpu
entry.load_package()
rope_ops = importlib.import_module("mlx_metal_kernels_b200.ops.rope_ops")
layer_ops = importlib.import_module("mlx_metal_kernels_b200.ops.decode_layer_ops")
EPS = 1e-6


def tables(R, length=64, theta=10000.0):
    return rope_ops.rotary_tables(rope_ops.RotaryConfig(head_dim=R, theta=theta), length)


def want64(x, weight, cos, sin, positions, layout):
    """(result in fp64, |u| + |v| of every element's pair, or the element's own magnitude) for x [T, H, D]."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.double()
    R = 2 * cos.shape[1]
    size = y.abs().clone()
    for i in range(R // 2):
        iu, iv = (i, i + R // 2) if layout == "half" else (2 * i, 2 * i + 1)
        ok = ((positions >= 0) & (positions < cos.shape[0])).reshape(-1, 1)
        at = positions.clamp(0, cos.shape[0] - 1).long()
        c = torch.where(ok, cos[at, i].double().reshape(-1, 1), torch.ones((), dtype=torch.float64))
        s = torch.where(ok, sin[at, i].double().reshape(-1, 1), torch.zeros((), dtype=torch.float64))
        u, v = y[..., iu].clone(), y[..., iv].clone()
        size[..., iu] = size[..., iv] = u.abs() + v.abs()
        y[..., iu], y[..., iv] = u * c - v * s, u * s + v * c
    return y, size


def assert_close(got, want, size, dtype, normed, D):
    """fp32: two products and a sum (3 roundings of values up to |u| + |v|); with a norm in front a sum of D squares (relative
    error at most D/2 steps, halved by the root), the root and three products.  Then one rounding to the type (smallest
    step of fp16: 2^-24)."""
    steps = 3 + (D / 2 + 6 if normed else 0)
    half = torch.finfo(dtype).eps / 2
    bound = half * want.abs() + (1 + half) * steps * 2.0 ** -24 * size + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= bound).all()), f"worst excess {float((err - bound).max())}"


SHAPES = [  # D, R, Hq, Hkv, T
    (128, 128, 32, 8, 5), (128, 64, 4, 4, 3), (128, 32, 7, 1, 2), (64, 64, 8, 2, 9), (64, 16, 3, 3, 1), (256, 256, 5, 1, 4),
    (256, 112, 2, 2, 3), (32, 32, 6, 2, 33), (80, 80, 4, 2, 5), (96, 48, 3, 1, 4), (128, 20, 4, 2, 3), (6, 2, 3, 1, 2), (7, 6, 2, 1, 3),
    (16, 16, 2, 2, 4), (512, 512, 2, 1, 2),
]


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,R,Hq,Hkv,T", SHAPES)
@pytest.mark.parametrize("normed", [False, True])
def test_rotation(cuda, D, R, Hq, Hkv, T, dtype, layout, normed):
    g = gen(D * R + T)
    qkv = torch.randn((T, Hq + 2 * Hkv, D), generator=g).to(dtype)
    q, k = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv]
    cos, sin = tables(R)
    positions = torch.randint(0, 64, (T,), generator=g, dtype=torch.int32)
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=g)).to(dtype) for _ in range(2)) if normed else (None, None)
    dev = qkv.to(cuda)
    args = (cos.to(cuda), sin.to(cuda), positions.to(cuda))
    strided = (dev[:, :Hq], dev[:, Hq:Hq + Hkv])

    def call(pair, **kw_):
        if normed:
            return rope_ops.head_norm_rope(*pair, qw.to(cuda), kw.to(cuda), *args, eps=EPS, layout=layout, **kw_)
        return rope_ops.apply_rope(*pair, *args, layout=layout, **kw_)

    got = call(strided)
    for x, w, y in ((q, qw, got[0]), (k, kw, got[1])):
        want, size = want64(x, w, cos, sin, positions, layout)
        assert y.is_contiguous() and y.shape == x.shape
        assert_close(y, want, size, dtype, normed, D)
    assert torch.equal(dev.cpu(), qkv)
    again = call(tuple(t.contiguous() for t in strided))
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    kept = dev[:, Hq + Hkv:].clone()
    back = call(strided, inplace=True)
    assert all(torch.equal(a, b) for a, b in zip(got, back)) and torch.equal(dev[:, :Hq], got[0])
    assert torch.equal(dev[:, Hq + Hkv:], kept)
    assert cabi.device_status() == 0


def test_shapes_of_prompts_and_single_tensors(cuda):
    B, S, H, D = 2, 7, 3, 64
    q = torch.randn((B, S, H, D), generator=gen(1)).to(torch.float16)
    cos, sin = tables(D)
    pos = torch.arange(S, dtype=torch.int64)
    got, none = rope_ops.apply_rope(q.to(cuda), None, cos.to(cuda), sin.to(cuda), pos.to(cuda))
    assert none is None and got.shape == q.shape
    want, size = want64(q.reshape(B * S, H, D), None, cos, sin, pos.repeat(B), "interleaved")
    assert_close(got.reshape(B * S, H, D), want, size, torch.float16, False, D)
    turned = q.to(cuda).transpose(0, 1)                       # leading dimensions of two strides: copied
    got2, _ = rope_ops.apply_rope(turned, None, cos.to(cuda), sin.to(cuda), pos.to(cuda).reshape(S, 1).expand(S, B))
    assert torch.equal(got2.transpose(0, 1), got)
    spread = q.to(cuda)[..., None].expand(B, S, H, D, 2)[..., 0]
    assert torch.equal(rope_ops.apply_rope(spread, None, cos.to(cuda), sin.to(cuda), pos.to(cuda))[0], got)
    odd = torch.zeros(B * S * H * D + 1, dtype=torch.float16, device=cuda)[1:].view(B, S, H, D)      # 2-byte alignment
    odd.copy_(q)
    assert torch.equal(rope_ops.apply_rope(odd, None, cos.to(cuda), sin.to(cuda), pos.to(cuda))[0], got)
    for shape in ((0, 3, 64), (2, 0, 3, 64)):
        empty = torch.zeros(shape, dtype=torch.float16, device=cuda)
        a, b = rope_ops.apply_rope(empty, empty, cos.to(cuda), sin.to(cuda), torch.zeros(shape[:-2], dtype=torch.int32, device=cuda))
        assert a.shape == b.shape == shape


@pytest.mark.parametrize("D", [64, 80])
def test_positions_outside_the_table(cuda, D):
    x = torch.randn((4, 2, D), generator=gen(2)).to(torch.bfloat16).to(cuda)
    cos, sin = (t.to(cuda) for t in tables(D, 16))
    positions = torch.tensor([-1, 16, 15, 2 ** 33], device=cuda)
    cabi.device_status()
    got, _ = rope_ops.apply_rope(x, None, cos, sin, positions)
    assert cabi.device_status() == 6 and cabi.device_status() == 0
    assert torch.equal(got[[0, 1, 3]], x[[0, 1, 3]]) and not torch.equal(got[2], x[2])


def test_values_that_are_not_finite_stay_in_their_heads(cuda):
    x = torch.randn((3, 4, 64), generator=gen(3)).to(torch.float16).to(cuda)
    cos, sin = (t.to(cuda) for t in tables(64))
    pos = torch.tensor([1, 2, 3], device=cuda, dtype=torch.int32)
    w = torch.ones(64, device=cuda)
    clean, _ = rope_ops.head_norm_rope(x, None, w, None, cos, sin, pos)
    x[1, 2, 5], x[0, 0, 0] = float("nan"), float("inf")
    got, _ = rope_ops.head_norm_rope(x, None, w, None, cos, sin, pos)
    same = torch.ones(3, 4, dtype=torch.bool, device=cuda)
    same[1, 2] = same[0, 0] = False
    assert torch.equal(got[same], clean[same]) and bool(got[1, 2].isnan().all()) and bool(got[0, 0].isnan().any())
    zero, _ = rope_ops.head_norm_rope(torch.zeros_like(x), None, w, None, cos, sin, pos)
    assert bool((zero == 0).all())


def test_strides_past_32_bits(cuda):
    """Rows further apart than 2^31 elements."""
    far = torch.empty(2 ** 31 + 4096, dtype=torch.float16, device=cuda)
    q = far.as_strided((2, 2, 64), (2 ** 31 + 2048, 64, 1))
    q.copy_(torch.randn((2, 2, 64), generator=gen(4)))
    cos, sin = (t.to(cuda) for t in tables(64))
    pos = torch.tensor([3, 9], device=cuda)
    assert torch.equal(rope_ops.apply_rope(q, None, cos, sin, pos)[0], rope_ops.apply_rope(q.contiguous(), None, cos, sin, pos)[0])


def make_cache(bits, pages, P, Hkv, D, G, table, lengths, device, seed):
    g = gen(seed)
    values = torch.randn((2, pages, P, Hkv, D), generator=g).to(torch.float16)
    dp = (D + 1) // 2 if bits == 4 else D
    codes = torch.randint(0, 256, (2, pages, P, Hkv, dp), generator=g, dtype=torch.int32).to(torch.uint8)
    scales = values[..., :-(-D // G)].abs().contiguous()
    return pq_ops.PagedQuantizedKVCache(
        k_pages_q=codes[0].to(device), v_pages_q=codes[1].to(device), k_scales=scales[0].to(device), v_scales=scales[1].to(device),
        block_table=table.to(device), lengths=lengths.to(device), bits=bits, page_size=P, group_size=G,
        original_page_shape=(pages, P, Hkv, D))


def tokens_of(starts, counts):
    seq = torch.cat([torch.full((n,), i, dtype=torch.int32) for i, n in enumerate(counts)])
    pos = torch.cat([torch.arange(s, s + n, dtype=torch.int32) for s, n in zip(starts, counts)])
    return seq, pos


@pytest.mark.parametrize("D,R,G,P,Hq,Hkv", [(128, 128, 32, 16, 8, 2), (128, 64, 64, 16, 4, 4), (64, 64, 64, 16, 5, 5), (256, 32, 16, 8, 2, 1),
                                            (128, 128, 128, 5, 4, 1), (32, 32, 8, 16, 3, 1), (80, 40, 20, 7, 2, 1), (128, 128, 48, 16, 2, 2),
                                            (36, 36, 5, 4, 2, 1)])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_quantised_append(cuda, D, R, G, P, Hq, Hkv, bits, layout, dtype):
    """Without norms the rows and their codes are fixed to the bit; nothing but the tokens' slots changes."""
    starts, counts = [0, P - 1, 2 * P + 1], [3, 2, 1]
    seq, pos = tokens_of(starts, counts)
    table = torch.tensor([[7, 2, -1, -1], [0, 5, -1, -1], [3, 1, 6, -1]], dtype=torch.int32)
    lengths = torch.tensor([s + n for s, n in zip(starts, counts)], dtype=torch.int32)
    cache = make_cache(bits, 8, P, Hkv, D, G, table, lengths, cuda, 5)
    before = {n: getattr(cache, n).cpu().clone() for n in ("k_pages_q", "v_pages_q", "k_scales", "v_scales")}
    T = len(seq)
    qkv = torch.randn((T, (Hq + 2 * Hkv) * D), generator=gen(6)).to(dtype)
    cos, sin = tables(R)
    got = layer_ops.norm_rope_kv_append(qkv.to(cuda), cos.to(cuda), sin.to(cuda), pos.to(cuda), cache, Hq, sequences=seq.to(cuda), layout=layout)
    rows = qkv.reshape(T, -1, D)
    want = []
    for x in (rows[:, :Hq], rows[:, Hq:Hq + Hkv]):
        y, size = want64(x, None, cos, sin, pos, layout)
        r = rope_ops.apply_rope(x.contiguous().to(cuda), None, cos.to(cuda), sin.to(cuda), pos.to(cuda), layout=layout)[0]
        assert_close(r, y, size, dtype, False, D)
        want.append(r.cpu())
    assert torch.equal(got.cpu(), want[0])
    for name, sname, x in (("k_pages_q", "k_scales", want[1]), ("v_pages_q", "v_scales", rows[:, Hq + Hkv:])):
        codes, scales = before[name], before[sname]
        for t in range(T):
            page, slot = int(table[seq[t], pos[t] // P]), int(pos[t] % P)
            c, s = quantise(x[t].float(), bits, G)
            codes[page, slot], scales[page, slot] = c, s
        assert torch.equal(getattr(cache, name).cpu(), codes), name
        assert torch.equal(getattr(cache, sname).cpu(), scales), sname
    assert cabi.device_status() == 0


def quantise(v, bits, G):
    """The append's rule on fp32 values [H, D], in 32 bits: codes (packed for 4 bits) and fp16 scales."""
    top, off = (127.0, 128) if bits == 8 else (7.0, 8)
    H, D = v.shape
    codes, scales = torch.zeros((H, D), dtype=torch.int32), torch.zeros((H, -(-D // G)))
    for g in range(-(-D // G)):
        x = v[:, g * G:(g + 1) * G]
        s = x.abs().amax(-1).clamp_min(1e-8) * (torch.tensor(1.0) / top)
        codes[:, g * G:(g + 1) * G] = (torch.round(x / s[:, None]).clamp(-top, top)).to(torch.int32) + off
        scales[:, g] = s
    if bits == 4:
        pad = torch.nn.functional.pad(codes, (0, D % 2))
        codes = pad[:, 0::2] | (pad[:, 1::2] << 4)
    return codes.to(torch.uint8), scales.to(torch.float16)


def assert_quantisers_agree(codes, scales, values, bits, G):
    """Codes [.., bytes] and scales of values [.., D] beside quantize_kv_pages': scales within a step of fp16, codes the same but for values
    exactly half way between two (2 limit |v| an odd multiple of the group's largest magnitude), which are one off."""
    want_codes, want_scales = pq_ops._quantize_groups(values.contiguous(), bits, G)
    gap = (scales.contiguous().view(torch.int16).int() - want_scales.view(torch.int16).int()).abs()
    assert int(gap.max()) <= 1
    if bits == 4:
        codes, want_codes = (torch.stack((c & 15, c >> 4), dim=-1).flatten(-2) for c in (codes, want_codes))
    off = codes.int() - want_codes.int()
    at = off != 0
    if bool(at.any()):
        v = values.double().unflatten(-1, (-1, G)).abs()
        top = v.amax(-1, keepdim=True)
        halves = (2 * (127 if bits == 8 else 7) * v / top).flatten(-2)[at]      # exact: few bits over few bits, were it an integer
        assert bool((off[at].abs() == 1).all()) and bool((halves % 2 == 1).all())


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("D,R,layout", [(128, 128, "half"), (128, 32, "half"), (64, 64, "interleaved"), (80, 80, "half")])
def test_append_with_norms(cuda, bits, D, R, layout):
    """The cached k lies within half a quantisation step of the formula's, beside the roundings of the row and of the scale."""
    P, Hq, Hkv, G, dtype = 16, 6, 3, 16, torch.bfloat16
    seq, pos = tokens_of([0, 20], [18, 5])
    table = torch.tensor([[4, 1], [0, 3]], dtype=torch.int32)
    T = len(seq)
    g = gen(8)
    qkv = torch.randn((T, (Hq + 2 * Hkv) * D), generator=g).to(dtype)
    qw, kw = (1 + 0.2 * torch.randn(D, generator=g)), (1 + 0.2 * torch.randn(D, generator=g)).to(dtype)
    cos, sin = tables(R)
    rows = qkv.reshape(T, -1, D)
    args = (qkv.to(cuda), cos.to(cuda), sin.to(cuda), pos.to(cuda))
    kwargs = dict(sequences=seq.to(cuda), q_weight=qw.to(cuda), k_weight=kw.to(cuda), eps=EPS, layout=layout)
    page, slot = table[seq.long(), (pos // P).long()].long(), (pos % P).long()
    if bits == 16:
        pages = torch.full((2, 6, P, Hkv, D), 7.0, dtype=dtype, device=cuda)
        got = pkv_ops.norm_rope_kv_append_pages(*args, pages[0], pages[1], table.to(cuda), Hq, **kwargs)
        held = pages.cpu()
        k, v = held[0][page, slot], held[1][page, slot]
        held[:, page, slot] = 7.0
        assert bool((held == 7.0).all())
        step = torch.zeros(T, Hkv, D, dtype=torch.float64)
    else:
        cache = make_cache(bits, 6, P, Hkv, D, G, table, torch.zeros(2, dtype=torch.int32), cuda, 9)
        got = layer_ops.norm_rope_kv_append(*args, cache, Hq, **kwargs)
        k, v = (t.cpu()[page, slot] for t in pq_ops.dequantize_kv_pages(cache))
        step = cache.k_scales.cpu()[page, slot].double().repeat_interleave(G, -1)
    want, size = want64(rows[:, :Hq], qw, cos, sin, pos, layout)
    assert_close(got, want, size, dtype, True, D)
    want, size = want64(rows[:, Hq:Hq + Hkv], kw, cos, sin, pos, layout)
    if bits == 16:
        assert_close(k, want, size, dtype, True, D)
        assert torch.equal(v, rows[:, Hq + Hkv:])
    else:
        # half a step; the row's own rounding; the scale's (fp16) on up to 127 or 7 steps; the dequantised fp16 value's
        top = 127 if bits == 8 else 7
        bound = step * (0.5 + 2 * top * 2.0 ** -11) + want.abs() * (2.0 ** -8 + 2.0 ** -11) + (D / 2 + 9) * 2.0 ** -23 * size
        assert bool(((k.double() - want).abs() <= bound).all())
    assert cabi.device_status() == 0


@pytest.mark.parametrize("D", [64, 80])
@pytest.mark.parametrize("bits", [8, 16])
def test_append_padding_and_missing_pages(cuda, D, bits):
    """Padding writes zeros to q and nothing else; tokens without a page append nothing and are reported."""
    P, Hq, Hkv = 4, 2, 1
    table = torch.tensor([[1, -1, 9], [0, 2, 3]], dtype=torch.int32, device=cuda)
    cos, sin = (t.to(cuda) for t in tables(D, 12))
    qkv = torch.randn((7, (Hq + 2 * Hkv) * D), generator=gen(11)).to(torch.float16).to(cuda)
    seq = torch.tensor([0, -1, 0, 0, 2, 1, 1], dtype=torch.int32, device=cuda)
    pos = torch.tensor([0, 10 ** 9, 5, 9, 0, -3, 11], dtype=torch.int32, device=cuda)       # only the first and the last have a page
    if bits == 16:
        pools = [torch.full((5, P, Hkv, D), 3.0, dtype=torch.float16, device=cuda) for _ in range(2)]
        call = lambda q, s, p: pkv_ops.norm_rope_kv_append_pages(q, cos, sin, p, *pools, table, Hq, sequences=s)
    else:
        cache = make_cache(8, 5, P, Hkv, D, D, table, torch.zeros(2, dtype=torch.int32), cuda, 12)
        pools = [cache.k_pages_q, cache.v_pages_q, cache.k_scales, cache.v_scales]
        call = lambda q, s, p: layer_ops.norm_rope_kv_append(q, cos, sin, p, cache, Hq, sequences=s)
    before = [t.clone() for t in pools]
    cabi.device_status()
    got = call(qkv, seq, pos)
    assert cabi.device_status() == 7
    assert bool((got[1] == 0).all())
    first_last = [t.clone() for t in pools]
    for t, b in zip(pools, before):
        t.copy_(b)
    part = call(qkv[[0, 6]], seq[[0, 6]].contiguous(), pos[[0, 6]].contiguous())
    assert cabi.device_status() == 0
    assert torch.equal(part, got[[0, 6]]) and all(torch.equal(a, b) for a, b in zip(first_last, pools))
    for t, b in zip(pools, before):
        changed = (t != b).reshape(5, P, -1).any(-1)
        changed[1, 0] = changed[3, 3] = False
        assert not bool(changed.any())
    empty = call(qkv[:0], seq[:0], pos[:0])
    assert empty.shape == (0, Hq, D)


def test_append_equals_the_decode_operator(cuda):
    """One new token of every sequence, interleaved, no norm: the same queries and, up to ties, the same cache as rope_kv_append."""
    B, Hq, Hkv, D, P = 5, 8, 2, 128, 16
    case = synth.paged_kv_case(B, Hkv, D, P, num_pages=40, min_len=20, max_len=90, bits=8, group_size=32, seed=3)
    qkv = synth.activations((B, (Hq + 2 * Hkv) * D), 4).to(cuda)
    cos, sin = (t.to(cuda) for t in tables(D, 128))
    pos = (case["lengths"] - 1).to(cuda)
    caches = [pq_ops.PagedQuantizedKVCache(**{k: (v.to(cuda) if torch.is_tensor(v) else v) for k, v in case.items()}) for _ in range(2)]
    a = layer_ops.rope_kv_append(qkv, cos, sin, pos, caches[0], Hq)
    wide = torch.zeros(B, qkv.shape[1] + 64, dtype=torch.float16, device=cuda)       # rows of a wider buffer
    wide[:, :-64] = qkv
    b = layer_ops.norm_rope_kv_append(wide[:, :-64], cos, sin, pos, caches[1], Hq)
    assert torch.equal(a, b)
    page, slot = table_rows(case["block_table"].to(cuda), pos, P)
    rows = qkv.reshape(B, -1, D)
    turned = rope_ops.apply_rope(rows[:, Hq:Hq + Hkv], None, cos, sin, pos)[0]
    for codes, scales, values in (("k_pages_q", "k_scales", turned), ("v_pages_q", "v_scales", rows[:, Hq + Hkv:])):
        assert_quantisers_agree(getattr(caches[1], codes)[page, slot], getattr(caches[1], scales)[page, slot], values, 8, 32)
        for n in (codes, scales):
            x, y = (getattr(c, n).clone() for c in caches)
            x[page, slot] = y[page, slot] = 0
            assert torch.equal(x, y)


def table_rows(table, pos, P):
    return table[torch.arange(len(pos), device=pos.device), (pos // P).long()].long(), (pos % P).long()


def test_streams_and_graphs(cuda):
    """On a stream of its own, and captured: a replay reads new rows and positions."""
    T, Hq, Hkv, D, P = 3, 4, 2, 128, 16
    cos, sin = (t.to(cuda) for t in tables(D, 64))
    w = (1 + 0.1 * torch.randn(D, generator=gen(13))).to(torch.float16).to(cuda)
    table = torch.arange(12, dtype=torch.int32, device=cuda).reshape(3, 4)
    pools = [torch.zeros((12, P, Hkv, D), dtype=torch.float16, device=cuda) for _ in range(2)]
    qkv = torch.randn((T, (Hq + 2 * Hkv) * D), generator=gen(14)).to(torch.float16).to(cuda)
    pos = torch.tensor([0, 17, 63], dtype=torch.int32, device=cuda)
    call = lambda: pkv_ops.norm_rope_kv_append_pages(qkv, cos, sin, pos, *pools, table, Hq, q_weight=w, k_weight=w, layout="half")
    want = call().clone()
    pages = [p.clone() for p in pools]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
        turned = rope_ops.head_norm_rope(qkv.view(T, -1, D)[:, :Hq], None, w, None, cos, sin, pos, layout="half")[0]
    side.synchronize()
    assert torch.equal(other, want) and torch.equal(turned, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    rows, at = qkv.clone(), pos.clone()
    qkv.copy_(torch.randn(qkv.shape, generator=gen(15)))
    pos.copy_(torch.tensor([5, 1, 40]))
    graph.replay()
    fresh = [p.clone() for p in pools]
    assert torch.equal(out, call()) and all(torch.equal(a, b) for a, b in zip(fresh, pools))
    qkv.copy_(rows)
    pos.copy_(at)
    graph.replay()
    assert torch.equal(out, want)
    for p, q in zip(pools, pages):
        for b in range(3):
            page, slot = int(table[b, at[b] // P]), int(at[b] % P)
            assert torch.equal(p[page, slot], q[page, slot])


def many(cuda):
    """Tokens from which on the ring kernel runs (eight per SM), and then some."""
    return 8 * torch.cuda.get_device_properties(cuda).multi_processor_count + 37


@pytest.mark.parametrize("D,R,Hq,Hkv", [(128, 128, 8, 2), (128, 64, 5, 3), (64, 64, 7, 1), (256, 32, 9, 2), (32, 32, 3, 0), (64, 16, 64, 8)])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_many_tokens(cuda, D, R, Hq, Hkv, layout, dtype):
    """Without norms the bits of calls of few tokens, in place too; with norms the formula's values."""
    T = many(cuda)
    g = gen(D + R)
    qkv = torch.randn((T, Hq + Hkv + 1, D), generator=g).to(dtype)
    pos = torch.randint(-3, 70, (T,), generator=g, dtype=torch.int32)
    cos, sin = tables(R)
    dev = qkv.to(cuda)
    q, k = dev[:, :Hq], dev[:, Hq:Hq + Hkv] if Hkv else None
    args = (cos.to(cuda), sin.to(cuda), pos.to(cuda))
    cabi.device_status()
    got = rope_ops.apply_rope(q, k, *args, layout=layout)
    assert cabi.device_status() == 6
    for x, y in ((q, got[0]), (k, got[1])):
        if x is not None:
            few = [rope_ops.apply_rope(x[i:i + 64], None, *args[:2], args[2][i:i + 64], layout=layout)[0] for i in range(0, T, 64)]
            assert torch.equal(y, torch.cat(few))
    w = (1 + 0.2 * torch.randn(D, generator=g))
    normed = rope_ops.head_norm_rope(q, k, w.to(cuda), None, *args, eps=EPS, layout=layout)
    want, size = want64(qkv[:, :Hq], w, cos, sin, pos, layout)
    assert_close(normed[0], want, size, dtype, True, D)
    if k is not None:
        assert torch.equal(normed[1], got[1])
    rest = dev[:, Hq + Hkv:].clone()
    rope_ops.apply_rope(q, k, *args, layout=layout, inplace=True)
    assert torch.equal(q, got[0]) and (k is None or torch.equal(k, got[1])) and torch.equal(dev[:, Hq + Hkv:], rest)
    assert cabi.device_status() == 6


@pytest.mark.parametrize("bits,D,R,G,layout", [(8, 128, 128, 32, "half"), (4, 128, 128, 32, "interleaved"), (8, 128, 64, 64, "half"), (4, 64, 32, 16, "half"),
                                               (8, 256, 256, 256, "interleaved"), (8, 128, 128, 8, "half"), (16, 128, 128, 32, "half"), (16, 64, 32, 8, "interleaved")])
def test_append_of_many_tokens(cuda, bits, D, R, G, layout):
    """The bits of appends of few tokens: rows, codes, scales, padding, tokens without a page, values that are not finite."""
    T, P, Hq, Hkv, dtype = many(cuda), 16, 6, 2, torch.bfloat16
    g = gen(bits + D)
    B, blocks = 5, (T + 4) // 5 // P + 2
    pages = B * blocks + 3
    order = torch.randperm(pages, generator=g)[:B * blocks].to(torch.int32).reshape(B, blocks)
    order[2, 1] = -1
    seq = torch.arange(T, dtype=torch.int32) % B
    pos = (torch.arange(T, dtype=torch.int32) // B) + 3
    seq[7::50] = -1
    seq[9] = B
    qkv = torch.randn((T, Hq + 2 * Hkv, D), generator=g).to(dtype)
    qkv[3, Hq, 5], qkv[4, Hq + 1, 0], qkv[5, Hq + Hkv, 1], qkv[6, Hq, 3] = float("nan"), float("inf"), float("-inf"), float("nan")
    qkv[8, Hq:] = 0.0
    qkv[10, Hq:] = 1e-12
    qkv = qkv.reshape(T, -1).to(cuda)
    cos, sin = (t.to(cuda) for t in tables(R, int(pos.max()) + 1))
    table, seq, pos = order.to(cuda), seq.to(cuda), pos.to(cuda)
    results = []
    for step in (T, 64):
        cache = make_cache(bits if bits < 16 else 8, pages, P, Hkv, D, G, order, torch.zeros(B, dtype=torch.int32), cuda, 7)
        plain = [torch.full((pages, P, Hkv, D), 2.0, dtype=dtype, device=cuda) for _ in range(2)]
        out = []
        for i in range(0, T, step):
            part = (qkv[i:i + step], cos, sin, pos[i:i + step])
            if bits == 16:
                out.append(pkv_ops.norm_rope_kv_append_pages(*part, *plain, table, Hq, sequences=seq[i:i + step], layout=layout))
            else:
                out.append(layer_ops.norm_rope_kv_append(*part, cache, Hq, sequences=seq[i:i + step], layout=layout))
        assert cabi.device_status() == 7
        pool = plain if bits == 16 else [cache.k_pages_q, cache.v_pages_q, cache.k_scales, cache.v_scales]
        results.append([torch.cat(out)] + pool)
    for a, b in zip(*results):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert bool((results[0][0][7::50] == 0).all())
    if bits < 16:                                            # and the quantiser's codes, also for what is not finite
        v = qkv.reshape(T, -1, D)[:, Hq + Hkv:]
        page, slot = table[seq.clamp(0, B - 1).long(), (pos // P).long()].long(), (pos % P).long()
        held = (seq >= 0) & (seq < B) & (page >= 0)
        assert_quantisers_agree(results[0][2][page[held], slot[held]], results[0][4][page[held], slot[held]], v[held], bits, G)


def test_captured_calls_of_many_tokens(cuda):
    """Two graphs over the ring kernel, replayed in turn on rows, positions and sequences that were not there at capture."""
    T, P, Hq, Hkv, D, B = many(cuda), 16, 4, 2, 128, 3
    blocks = T // B // P + 3
    table = torch.randperm(B * blocks, generator=gen(41)).to(torch.int32).reshape(B, blocks).to(cuda)
    cos, sin = (t.to(cuda) for t in tables(D, blocks * P))
    w = (1 + 0.1 * torch.randn(D, generator=gen(42))).to(torch.bfloat16).to(cuda)
    pools = [torch.zeros((B * blocks, P, Hkv, D), dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    qkv = torch.randn((T, (Hq + 2 * Hkv) * D), generator=gen(43)).to(torch.bfloat16).to(cuda)
    seq = (torch.arange(T, dtype=torch.int32) % B).to(cuda)
    pos = (torch.arange(T, dtype=torch.int32) // B).to(cuda)
    calls = (lambda: pkv_ops.norm_rope_kv_append_pages(qkv, cos, sin, pos, *pools, table, Hq, sequences=seq, q_weight=w, k_weight=w),
             lambda: rope_ops.apply_rope(qkv.view(T, -1, D)[:, :Hq], None, cos, sin, pos)[0])
    for call in calls:
        call()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for call in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call())
    qkv.copy_(torch.randn(qkv.shape, generator=gen(44)))
    pos.copy_(pos.flip(0).clone())
    seq.copy_(seq.flip(0).clone())
    seq[5::40] = -1
    for p in pools:
        p.zero_()
    for graph in graphs + graphs:
        graph.replay()
    replayed = [p.clone() for p in pools]
    for p in pools:
        p.zero_()
    assert all(torch.equal(out, call()) for out, call in zip(outs, calls)) and all(torch.equal(a, b) for a, b in zip(replayed, pools))
    assert bool((outs[0][5::40] == 0).all()) and cabi.device_status() == 0
