"""GPU adapters against the formula in 64 bits."""
import importlib

import pytest
import torch

import __graft_entry__ as entry
from helpers import cabi, gen, mlp_ops, synth

pytestmark = pytest.mark.gpu
entry.load_package()
lora = importlib.import_module("mlx_metal_kernels_b200.ops.lora_ops")


def make(L, R, K, N, dtype, cuda, seed, ranks=None, scaling=True):
    g = gen(seed)
    a = (torch.randn((L, R, K), generator=g) * K ** -0.5).to(dtype).to(cuda)
    b = (torch.randn((L, N, R), generator=g) * 0.3).to(dtype).to(cuda)
    s = (0.5 + torch.rand(L, generator=g)).to(cuda) if scaling else None
    return lora.LoraAdapters(a, b, s, None if ranks is None else torch.tensor(ranks, dtype=torch.int32, device=cuda))


def check(got, y, x, ad, ids):
    """A sum of K fp32 products, 16 or more at a time (depth K/16 + 8, 2^-23 of the absolute sum per addition: tensor cores cut off),
    then of R products of values held to 2^-20 or better, then one rounding of the sum with y; fp16 results end at 2^-25."""
    rows, K = x.shape
    L, R, _ = ad.a.shape
    dtype = got.dtype
    ids = ids.long()
    some = ((ids >= 0) & (ids < L)).nonzero().reshape(-1)
    assert torch.equal(got[ids < 0], y[ids < 0])
    if some.numel() == 0:
        return
    l = ids[some]
    a, b, xs = ad.a[l].double(), ad.b[l].double(), x[some].double()
    if ad.ranks is not None:
        keep = (torch.arange(R, device=x.device)[None] < ad.ranks[l][:, None])
        a = torch.where(keep[:, :, None], a, torch.zeros_like(a))
        b = torch.where(keep[:, None, :], b, torch.zeros_like(b))
    s = ad.scaling[l].double()[:, None] if ad.scaling is not None else 1.0
    low = torch.einsum("trk,tk->tr", a, xs)
    low_err = (K / 16 + 8) * 2.0 ** -23 * torch.einsum("trk,tk->tr", a.abs(), xs.abs()) + 2.0 ** -20 * low.abs().amax(-1, keepdim=True)
    delta = s * torch.einsum("tnr,tr->tn", b, low)
    err = s * (torch.einsum("tnr,tr->tn", b.abs(), low_err) + (R + 4) * 2.0 ** -23 * torch.einsum("tnr,tr->tn", b.abs(), low.abs()))
    want = y[some].double() + delta
    half = torch.finfo(dtype).eps / 2
    bound = half * want.abs() + (1 + half) * (err + 2.0 ** -23 * want.abs()) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    off = (got[some].double() - want).abs()
    assert bool((off <= bound).all()), f"worst excess {float((off - bound).max())}, of {float(bound.mean())}"


SHAPES = [  # rows, N, K, L, R
    (1, 256, 512, 1, 16), (1, 4096, 4096, 4, 16), (4, 512, 1024, 3, 8), (16, 384, 640, 5, 32), (17, 320, 256, 2, 64), (33, 1000, 520, 7, 24),
    (40, 136, 2592, 40, 16), (64, 5003, 96, 3, 12), (5, 77, 33, 2, 3), (2, 8, 8, 2, 1), (100, 256, 512, 1, 128), (7, 512, 264, 3, 100),
    (130, 2048, 1024, 4, 16), (300, 520, 512, 3, 64), (3, 264, 70000, 2, 16), (20, 1, 64, 2, 16), (9, 24, 64, 2, 200), (18, 96, 128, 2, 160),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,N,K,L,R", SHAPES)
@pytest.mark.parametrize("spread", ["mixed", "runs"])
def test_lora_add(cuda, rows, N, K, L, R, dtype, spread):
    g = gen(rows * N + R)
    x = torch.randn((rows, K), generator=g).to(dtype).to(cuda)
    y = torch.randn((rows, N), generator=g).to(dtype).to(cuda)
    ids = torch.randint(-1, L, (rows,), generator=g, dtype=torch.int32)
    if spread == "runs":
        ids = (torch.arange(rows) // 21 % L).to(torch.int32)
    ranks = torch.randint(0, R + 1, (L,), generator=g).tolist() if spread == "mixed" else None
    if ranks:
        ranks[0] = R
    ad = make(L, R, K, N, dtype, cuda, rows + K, ranks, scaling=spread == "mixed")
    got = lora.lora_add(y, x, ad, ids.to(cuda))
    check(got, y, x, ad, ids.to(cuda))
    assert torch.equal(got, lora.lora_add(y, x, ad, ids.to(cuda)))          # the same bits again
    assert cabi.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,N,K,L,R", [(8, 6144, 96, 1, 40), (32, 6144, 256, 1, 64), (32, 6149, 64, 2, 64), (40, 6144, 64, 1, 24),
                                          (128, 4100, 128, 3, 256), (200, 8200, 64, 2, 16), (270, 8192, 40, 1, 128)])
@pytest.mark.parametrize("spread", ["mixed", "runs"])
def test_many_rows_of_few_adapters(cuda, rows, N, K, L, R, dtype, spread):
    """Fewer groups of rows than clusters: several share a group's columns."""
    test_lora_add(cuda, rows, N, K, L, R, dtype, spread)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rows,N,K,G", [(1, 512, 1024, 64), (6, 1003, 96, 32), (40, 256, 512, 64)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_quantized_linear(cuda, bits, rows, N, K, G, dtype):
    """One rounding of the sum: off by at most the shared product's own rounding from the adapters added to that."""
    w, s, z = (t.to(cuda) for t in synth.quantized_weight(N, K, bits, G, seed=N))
    x = synth.activations((rows, K), 2).to(dtype).to(cuda)
    ids = torch.tensor([(i % 4) - 1 for i in range(rows)], dtype=torch.int32, device=cuda)
    ad = make(3, 16, K, N, dtype, cuda, 3)
    half = torch.finfo(dtype).eps / 2
    base = mlp_ops.quantized_linear(x, w, s, z, bits=bits, group_size=G)
    zero = torch.zeros_like(base)
    for residual in (None, synth.activations((rows, N), 5).to(dtype).to(cuda)):
        got = lora.lora_quantized_linear(x, w, s, z, ad, ids, bits=bits, group_size=G, residual=residual)
        low = lora.lora_add(zero, x, ad, ids)                # rounded: off by half a step of itself
        check(low, zero, x, ad, ids)
        want = base.double() + low.double() + (0.0 if residual is None else residual.double())
        bound = half * (want.abs() * (1 + 4 * half) + (base.double().abs() + low.double().abs()) * (1 + 4 * half)) + 2.0 ** -22 * (base.double().abs() + low.double().abs()) + 2.0 ** -24
        assert bool(((got.double() - want).abs() <= bound).all())
        if residual is None:
            assert torch.equal(got[ids < 0], base[ids < 0])


def test_shapes_of_prompts(cuda):
    B, S, K, N = 2, 5, 128, 64
    w, s, z = (t.to(cuda) for t in synth.quantized_weight(N, K, 4, 32, seed=1))
    ad = make(3, 8, K, N, torch.float16, cuda, 2)
    x = synth.activations((B, S, K), 3).to(cuda)
    per_sequence = torch.tensor([2, -1], device=cuda)                        # int64, one per sequence
    got = lora.lora_quantized_linear(x, w, s, z, ad, per_sequence, group_size=32)
    flat = lora.lora_quantized_linear(x.reshape(B * S, K), w, s, z, ad, per_sequence.repeat_interleave(S), group_size=32)
    assert got.shape == (B, S, N) and torch.equal(got.reshape(B * S, N), flat)
    turned = x.transpose(0, 1)
    ids = torch.tensor([[0, 1]] * S, device=cuda, dtype=torch.int32)
    again = lora.lora_quantized_linear(turned, w, s, z, ad, ids, group_size=32)
    want = lora.lora_quantized_linear(turned.contiguous(), w, s, z, ad, ids.contiguous(), group_size=32)
    assert torch.equal(again, want)
    assert lora.lora_quantized_linear(x[:0], w, s, z, ad, ids[:0, :1].expand(0, S), group_size=32).shape == (0, S, N)
    strided = lora.LoraAdapters(ad.a.transpose(1, 2).contiguous().transpose(1, 2), ad.b, ad.scaling)
    assert torch.equal(lora.lora_quantized_linear(x, w, s, z, strided, per_sequence, group_size=32), got)
    odd = torch.empty(ad.a.numel() + 1, dtype=torch.float16, device=cuda)[1:].view(ad.a.shape)      # 2-byte alignment
    odd.copy_(ad.a)
    y = torch.zeros(B * S, N, dtype=torch.float16, device=cuda)
    check(lora.lora_add(y, x.reshape(B * S, K), lora.LoraAdapters(odd, ad.b, ad.scaling), ids.reshape(-1)), y, x.reshape(B * S, K), ad, ids.reshape(-1))


def test_adapters_that_do_not_exist(cuda):
    x, y = torch.randn((3, 64), generator=gen(1)).half().to(cuda), torch.randn((3, 32), generator=gen(2)).half().to(cuda)
    ad = make(2, 16, 64, 32, torch.float16, cuda, 3)
    cabi.device_status()
    got = lora.lora_add(y, x, ad, torch.tensor([0, 2, 2 ** 40], device=cuda))
    assert cabi.device_status() == 10 and cabi.device_status() == 0
    assert torch.equal(got[1:], y[1:])
    assert torch.equal(got[:1], lora.lora_add(y[:1], x[:1], ad, torch.tensor([0], device=cuda)))


def test_unused_ranks_are_not_read(cuda):
    """NaN behind an adapter's rank, in adapters that no row uses, and in rows of other adapters."""
    K, N, R = 512, 256, 32
    ad = make(4, R, K, N, torch.float16, cuda, 4, ranks=[12, 0, 32, 5])
    x = torch.randn((20, K), generator=gen(5)).half().to(cuda)
    y = torch.randn((20, N), generator=gen(6)).half().to(cuda)
    ids = torch.tensor([0, 1, 3, -1] * 5, dtype=torch.int32, device=cuda)
    clean = lora.lora_add(y, x, ad, ids)
    check(clean, y, x, ad, ids)
    for l, rank in enumerate((12, 0, 0, 5)):
        ad.a[l, rank:] = float("nan")
        ad.b[l, :, rank:] = float("nan")
    assert torch.equal(lora.lora_add(y, x, ad, ids), clean)
    x[1], x[3], x[6] = float("nan"), float("inf"), float("inf")              # rows without rank, without adapter, and of adapter 3
    got = lora.lora_add(y, x, ad, ids)
    same = torch.ones(20, dtype=torch.bool, device=cuda)
    same[6] = False
    assert torch.equal(got[same], clean[same]) and not bool(got[6].isfinite().all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_large_and_small_values_between_the_factors(cuda, dtype):
    """A x far outside fp16's range, and far below its steps."""
    K, N, R = 256, 64, 16
    for size in (2.0 ** 12, 2.0 ** -20):
        ad = make(2, R, K, N, dtype, cuda, 7)
        ad.a[:] = (ad.a.float() * 16 * size ** 0.5).to(dtype)
        ad.b[:] = (ad.b.float() * 2.0 ** -8 / size).clamp(-6e4, 6e4).to(dtype)
        x = (torch.randn((5, K), generator=gen(8)) * 16 * size ** 0.5).to(dtype).to(cuda)
        y = torch.zeros((5, N), dtype=dtype, device=cuda)
        ids = torch.tensor([0, 1, 0, 1, -1], dtype=torch.int32, device=cuda)
        check(lora.lora_add(y, x, ad, ids), y, x, ad, ids)


def test_offsets_past_32_bits(cuda):
    """Factors behind the first 2^31 elements of the stack."""
    L, R, K, N = 540, 64, 64000, 32
    a = torch.empty((L, R, K), dtype=torch.float16, device=cuda)
    small = make(1, R, K, N, torch.float16, cuda, 9)
    a[L - 1] = small.a[0]
    b = torch.zeros((L, N, R), dtype=torch.float16, device=cuda)
    b[L - 1] = small.b[0]
    x, y = torch.randn((2, K), generator=gen(10)).half().to(cuda), torch.randn((2, N), generator=gen(11)).half().to(cuda)
    got = lora.lora_add(y, x, lora.LoraAdapters(a, b), torch.tensor([L - 1, -1], device=cuda))
    assert torch.equal(got, lora.lora_add(y, x, lora.LoraAdapters(small.a, small.b), torch.tensor([0, -1], device=cuda)))


def test_streams_and_graphs(cuda):
    """Captured once, replayed over other rows and ids; two graphs in turn; a stream of its own."""
    K, N = 1024, 512
    w, s, z = (t.to(cuda) for t in synth.quantized_weight(N, K, 4, 64, seed=1))
    ad = make(6, 16, K, N, torch.float16, cuda, 12)
    x = synth.activations((8, K), 3).to(cuda)
    ids = torch.tensor([0, 1, 2, 3, 4, 5, -1, 0], dtype=torch.int32, device=cuda)
    call = lambda: lora.lora_quantized_linear(x, w, s, z, ad, ids, group_size=64)
    want = call().clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
    side.synchronize()
    assert torch.equal(other, want)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(call())
    x.copy_(synth.activations((8, K), 4))
    ids.copy_(torch.tensor([5, 5, -1, 0, 0, 1, 2, 3]))
    fresh = call().clone()
    for graph in graphs + graphs:
        graph.replay()
    assert torch.equal(outs[0], fresh) and torch.equal(outs[1], fresh) and not torch.equal(fresh, want)


@pytest.mark.parametrize("R,ranks", [(24, (13, 0, 8)), (64, (33, 5, 64)), (136, (71, 1, 130))])
@pytest.mark.parametrize("N,rows", [(6144, 12), (200, 40)])
def test_values_behind_the_ranks_of_wide_factors(cuda, R, ranks, N, rows):
    """What lies behind an adapter's rank, NaN here, stays out of the products, wherever the rank ends in a piece of eight."""
    K = 96
    ad = make(3, R, K, N, torch.bfloat16, cuda, R, list(ranks))
    x = torch.randn((rows, K), generator=gen(21)).to(torch.bfloat16).to(cuda)
    y = torch.randn((rows, N), generator=gen(22)).to(torch.bfloat16).to(cuda)
    ids = (torch.arange(rows, dtype=torch.int32, device=cuda) % 4) - 1
    clean = lora.lora_add(y, x, ad, ids)
    check(clean, y, x, ad, ids)
    for l, rank in enumerate(ranks):
        ad.a[l, rank:] = float("nan")
        ad.b[l, :, rank:] = float("nan")
    assert torch.equal(lora.lora_add(y, x, ad, ids), clean)


@pytest.mark.parametrize("K,R", [(64, 8), (63, 8)])
def test_thousands_of_rows_and_results_in_place(cuda, K, R):
    """Many windows of rows, one CTA per cluster; the C call with out = y."""
    rows, N, L = 5000, 72, 6
    ad = make(L, R, K, N, torch.float16, cuda, 31)
    x = torch.randn((rows, K), generator=gen(32)).half().to(cuda)
    y = torch.randn((rows, N), generator=gen(33)).half().to(cuda)
    ids = torch.randint(-1, L, (rows,), generator=gen(34), dtype=torch.int32).to(cuda)
    got = lora.lora_add(y, x, ad, ids)
    check(got, y, x, ad, ids)
    lib = cabi.load()
    ws = torch.empty(lib.b200q_lora_workspace_bytes(rows, R), dtype=torch.uint8, device=cuda)
    cabi.check(lib.b200q_lora_add(x.data_ptr(), y.data_ptr(), y.data_ptr(), ad.a.data_ptr(), ad.b.data_ptr(), ad.scaling.data_ptr(), None,
                                  ids.data_ptr(), rows, N, K, L, R, cabi.F16, ws.data_ptr(), ws.numel(), cabi.stream()), "b200q_lora_add")
    assert torch.equal(y, got)


def exact_delta(x, ad, ids):
    """scaling B (A x) in 64 bits, 0 without an adapter, and what fp32 sums may be off: K and then R products one after the other, 2^-24 of the
    absolute sum each, the scaling, and the first sums' errors through B."""
    rows, K = x.shape
    L, R, _ = ad.a.shape
    out = torch.zeros((rows, ad.b.shape[1]), dtype=torch.float64, device=x.device)
    err = torch.zeros_like(out)
    for t, l in enumerate(ids.tolist()):
        if not 0 <= l < L:
            continue
        rank = R if ad.ranks is None else int(ad.ranks[l])
        a, b, s = ad.a[l, :rank].double(), ad.b[l, :, :rank].double(), 1.0 if ad.scaling is None else float(ad.scaling[l])
        low, low_abs = a @ x[t].double(), a.abs() @ x[t].double().abs()
        out[t] = s * (b @ low)
        err[t] = s * (b.abs() @ (K * 2.0 ** -24 * low_abs + (R + 4) * 2.0 ** -24 * low.abs()))
    return out, err


FEW = [  # rows, N, K, G, R
    (1, 512, 1024, 64, 16), (1, 4096, 4096, 64, 16), (2, 1003, 2592, 32, 12), (3, 777, 512, 128, 5), (4, 640, 1056, 32, 8), (4, 148, 96, 32, 32),
    (1, 100, 4096, 128, 32), (2, 5, 64, 32, 1), (1, 264, 14336, 64, 8), (4, 300, 8192, 64, 16),
]


@pytest.mark.parametrize("rows,N,K,G,R", FEW)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fused", [0, 1, -1])
def test_few_rows_beside_a_projection(cuda, bits, rows, N, K, G, R, dtype, fused):
    """Off by the roundings of the sum and of the plain product it is compared with, and by what fp32 sums lose: in one launch and in two,
    with residuals, rows without an adapter, an adapter that does not exist, and NaN behind the ranks."""
    w, s, z = (t.to(cuda) for t in synth.quantized_weight(N, K, bits, G, seed=N))
    x = synth.activations((rows, K), 2).to(dtype).to(cuda)
    ranks = [R, max(R - 3, 0), R // 2]
    ad = make(3, R, K, N, dtype, cuda, 3, ranks)
    for l, rank in enumerate(ranks):
        ad.a[l, rank:] = float("nan")
        ad.b[l, :, rank:] = float("nan")
    half = torch.finfo(dtype).eps / 2
    base = mlp_ops.quantized_linear(x, w, s, z, bits=bits, group_size=G)
    cabi.device_status()
    cabi.set_tuning("lora.fused", fused)
    try:
        for first in (-1, 0, 1, 2):
            ids = ((torch.arange(rows, dtype=torch.int32, device=cuda) + first + 1) % 4) - 1
            delta, err = exact_delta(x, ad, ids)
            for residual in (None, synth.activations((rows, N), 5).to(dtype).to(cuda)):
                got = lora.lora_quantized_linear(x, w, s, z, ad, ids, bits=bits, group_size=G, residual=residual)
                assert torch.equal(got, lora.lora_quantized_linear(x, w, s, z, ad, ids, bits=bits, group_size=G, residual=residual))
                rest = 0.0 if residual is None else residual.double()
                want = base.double() + delta + rest
                size = base.double().abs() + delta.abs() + (0.0 if residual is None else rest.abs())
                bound = half * (1 + 4 * half) * (want.abs() + base.double().abs()) + (1 + half) * err + 2.0 ** -22 * size + 2.0 ** -24
                assert bool(((got.double() - want).abs() <= bound).all())
                if residual is None:
                    assert torch.equal(got[ids < 0], base[ids < 0])
        assert cabi.device_status() == 0
        missing = torch.full((rows,), 3, dtype=torch.int32, device=cuda)
        assert torch.equal(lora.lora_quantized_linear(x, w, s, z, ad, missing, bits=bits, group_size=G), base)
        assert cabi.device_status() == 10
    finally:
        cabi.set_tuning("lora.fused", 0)


def test_few_rows_captured(cuda):
    """One launch, captured: a replay reads new rows, ids, ranks and scalings."""
    K, N = 2048, 768
    w, s, z = (t.to(cuda) for t in synth.quantized_weight(N, K, 4, 64, seed=1))
    ad = make(4, 8, K, N, torch.bfloat16, cuda, 12, [8, 3, 0, 5])
    x = synth.activations((2, K), 3).to(torch.bfloat16).to(cuda)
    ids = torch.tensor([1, -1], dtype=torch.int32, device=cuda)
    call = lambda: lora.lora_quantized_linear(x, w, s, z, ad, ids, group_size=64)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    x.copy_(synth.activations((2, K), 4))
    ids.copy_(torch.tensor([3, 0]))
    ad.ranks.copy_(torch.tensor([2, 3, 0, 8]))
    ad.scaling.mul_(2.0)
    graph.replay()
    assert torch.equal(out, call())
