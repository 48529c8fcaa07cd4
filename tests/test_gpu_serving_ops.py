"""The operators as a serving loop uses them together: projections with adapters, head norms with rotation and append, decode attention,
and pages reserved, forked, released and compacted under it."""
import importlib
import threading

import pytest
import torch

import __graft_entry__ as entry
from helpers import cabi, gen, pq_ops, synth

pytestmark = pytest.mark.gpu
entry.load_package()
lora = importlib.import_module("mlx_metal_kernels_b200.ops.lora_ops")
pages = importlib.import_module("mlx_metal_kernels_b200.ops.kv_page_ops")
rope_ops = importlib.import_module("mlx_metal_kernels_b200.ops.rope_ops")
layer_ops = importlib.import_module("mlx_metal_kernels_b200.ops.decode_layer_ops")

K, HQ, HKV, D, P, G = 512, 8, 2, 128, 16, 32
LAYERS, B, BLOCKS, POOL = 2, 5, 8, 40


class Loop:
    """Weights, adapters and caches of two small layers, one table for both."""

    def __init__(self, cuda, bits):
        N = (HQ + 2 * HKV) * D
        self.weights = [[t.to(cuda) for t in synth.quantized_weight(N, K, 4, 64, seed=20 + i)] for i in range(LAYERS)]
        g = gen(30)
        self.adapters = [lora.LoraAdapters((torch.randn((3, 16, K), generator=g) * K ** -0.5).half().to(cuda), (torch.randn((3, N, 16), generator=g) * 0.3).half().to(cuda),
                                           torch.tensor([0.5, 1.0, 2.0], device=cuda)) for _ in range(LAYERS)]
        self.norms = [[(1 + 0.1 * torch.randn(D, generator=g)).half().to(cuda) for _ in range(2)] for _ in range(LAYERS)]
        config = rope_ops.RotaryConfig(head_dim=D, theta=500000.0, scaling="llama3", factor=8.0, original_length=64)
        self.cos, self.sin = rope_ops.rotary_tables(config, BLOCKS * P, cuda)
        self.table = torch.full((B, BLOCKS), -1, dtype=torch.int32, device=cuda)
        self.lengths = torch.zeros(B, dtype=torch.int32, device=cuda)
        self.pool = pages.PagePool.empty(POOL, P, cuda)
        dp = D // 2 if bits == 4 else D
        z = lambda d, t: torch.zeros((POOL, P, HKV, d), dtype=t, device=cuda)
        self.caches = [pq_ops.PagedQuantizedKVCache(z(dp, torch.uint8), z(dp, torch.uint8), z(D // G, torch.float16), z(D // G, torch.float16), self.table,
                                                    self.lengths, bits=bits, page_size=P, group_size=G, original_page_shape=(POOL, P, HKV, D))
                       for _ in range(LAYERS)]

    def project(self, layer, x, ids):
        w, s, z = self.weights[layer]
        return lora.lora_quantized_linear(x, w, s, z, self.adapters[layer], ids, bits=4, group_size=64)

    def append(self, layer, qkv, positions, sequences=None):
        qw, kw = self.norms[layer]
        return layer_ops.norm_rope_kv_append(qkv, self.cos, self.sin, positions, self.caches[layer], HQ, sequences=sequences, q_weight=qw, k_weight=kw,
                                             layout="half")

    def attend(self, layer, q):
        return pq_ops.paged_quantized_kv_gqa_decode_attention(q.reshape(B, 1, HQ, D), self.caches[layer], backend="cuda")


@pytest.mark.parametrize("bits", [4, 8])
def test_a_serving_loop(cuda, bits):
    """Forked, compacted and captured: bit for bit what sequences of their own give that saw the same rows."""
    one, other = Loop(cuda, bits), Loop(cuda, bits)
    cabi.device_status()
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda)
    prompt = [37, 16, 0, 0, 5]                               # rows 2 and 3 will be children of 0 and 1
    seq = torch.cat([torch.full((n,), b, dtype=torch.int32) for b, n in enumerate(prompt)]).to(cuda)
    pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in prompt]).to(cuda)
    x = synth.activations((len(seq), K), 40).to(cuda)
    ids = ints(2, -1, 0, 1, 1)[seq.long()].contiguous()
    pages.reserve_pages(one.pool, one.table, one.lengths, ints(*prompt))
    rows = [one.project(i, x, ids) for i in range(LAYERS)]
    for i in range(LAYERS):
        one.append(i, rows[i], pos, seq)
    one.lengths += ints(*prompt)
    pages.fork_sequences(one.caches, one.pool, one.table, one.lengths, ints(0, 1), ints(2, 3))
    # the other world: every sequence on pages of its own, with its parent's rows where it has one
    origin = [0, 1, 0, 1, 4]
    full = [prompt[o] for o in origin]
    pages.reserve_pages(other.pool, other.table, other.lengths, ints(*full))
    pick = torch.cat([(seq == o).nonzero().reshape(-1) for o in origin])
    own = torch.cat([torch.full((n,), b, dtype=torch.int32) for b, n in enumerate(full)]).to(cuda)
    for i in range(LAYERS):
        other.append(i, rows[i][pick].contiguous(), pos[pick].contiguous(), own)
    other.lengths += ints(*full)
    assert torch.equal(one.lengths, other.lengths)
    assert int((one.pool.ref_counts > 0).sum()) == 6 and int((other.pool.ref_counts > 0).sum()) == 9      # 3 + 1 + 1 held once, and one copied page

    step_ids, h = ints(2, -1, 0, 1, 1), torch.zeros((B, K), dtype=torch.float16, device=cuda)

    def step(w, rows_out):
        pages.reserve_pages(w.pool, w.table, w.lengths, 1)
        positions = w.lengths.clone()
        w.lengths += 1
        outs = []
        for i in range(LAYERS):
            if rows_out[i] is None:
                rows_out[i] = w.project(i, h, step_ids)
            outs.append(w.attend(i, w.append(i, rows_out[i], positions)))
        return outs

    graph, shared = torch.cuda.CUDAGraph(), [None] * LAYERS
    table, lengths, counts = one.table.clone(), one.lengths.clone(), one.pool.ref_counts.clone()
    with torch.cuda.graph(graph):
        captured = step(one, shared)
    one.table.copy_(table)
    one.lengths.copy_(lengths)
    one.pool.ref_counts.copy_(counts)
    for n in range(14):                                      # over page borders
        h.copy_(synth.activations((B, K), 50 + n))
        graph.replay()
        want = step(other, list(shared))
        for a, b in zip(captured, want):
            assert torch.equal(a, b), n
        if n == 6:                                           # a parent ends and the pool is compacted, between two replays
            pages.release_sequences(one.pool, one.table, one.lengths, ints(0))
            pages.release_sequences(other.pool, other.table, other.lengths, ints(0))
            held = int((one.pool.ref_counts > 0).sum())
            remap = pages.compact_pages(one.caches, one.pool, one.table)
            assert int(remap.max()) == held - 1 and int((one.pool.ref_counts[:held] > 0).sum()) == held
    assert cabi.device_status() == 0
    assert torch.equal(shared[0], one.project(0, h, step_ids))
    # the formula, for one sequence and layer: softmax over the dequantised rows
    i, b = 1, 2
    k, v = pq_ops.dequantize_kv_pages(one.caches[i])
    n = int(one.lengths[b])
    at = torch.arange(n, device=cuda)
    page = one.table[b, at // P].long()
    k, v = (t[page, at % P].double() for t in (k, v))
    q = rope_ops.head_norm_rope(shared[i].reshape(B, -1, D)[:, :HQ], None, one.norms[i][0], None, one.cos, one.sin, one.lengths - 1, layout="half")[0][b].double()
    group = HQ // HKV
    scores = torch.einsum("hd,nhd->hn", q, k.repeat_interleave(group, 1)) / D ** 0.5
    want = torch.einsum("hn,nhd->hd", scores.softmax(-1), v.repeat_interleave(group, 1))
    # fp16 probabilities and output of the attention kernel: as its own parity tests allow
    assert float((captured[i][b, 0].double() - want).abs().max()) <= 2e-3 * float(want.abs().max().clamp_min(1.0))


def test_two_host_threads(cuda):
    """The same kernels launched by two threads with other sizes of shared memory, each on a stream of its own."""
    T = 8 * torch.cuda.get_device_properties(cuda).multi_processor_count + 5
    jobs = []
    for heads, R in ((4, 64), (24, 256)):
        g = gen(heads)
        x = torch.randn((T, heads, D), generator=g).half().to(cuda)
        cos, sin = rope_ops.rotary_tables(rope_ops.RotaryConfig(head_dim=D), 64, cuda)
        pos = (torch.arange(T) % 64).to(cuda)                              # int64: through the Python body, which lets go of the interpreter
        a, b = torch.randn((2, R, K), generator=g).half().to(cuda), (torch.randn((2, 640, R), generator=g) * 0.1).half().to(cuda)
        rows, y = torch.randn((20, K), generator=g).half().to(cuda), torch.randn((20, 640), generator=g).half().to(cuda)
        ids = (torch.arange(20, dtype=torch.int32) % 3 - 1).to(cuda)
        jobs.append(lambda x=x, cos=cos, sin=sin, pos=pos, a=a, b=b, rows=rows, y=y, ids=ids:
                    (rope_ops.apply_rope(x, None, cos, sin, pos)[0], lora.lora_add(y, rows, lora.LoraAdapters(a, b), ids)))
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    wrong = []

    def run(job, expected):
        try:
            with torch.cuda.device(cuda), torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(150):
                    got = job()
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(p, q) for p, q in zip(got, expected)):
                    wrong.append("results")
        except Exception as e:                                             # noqa: BLE001 - shown by the assertion below
            wrong.append(repr(e))

    threads = [threading.Thread(target=run, args=pair) for pair in zip(jobs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == [] and cabi.device_status() == 0
