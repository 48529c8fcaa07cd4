"""Operators around the quantised projections and the paged key/value cache, as measurable cases.

Five kinds of call that a serving program makes between the ones that perf/cases.py measures:

* lora    - a quantised projection with a low-rank adapter per row: y[t] = W x[t] + s[l] B[l] (A[l] x[t]), l = ids[t]
* rope    - queries and keys turned by their positions (interleaved or half layout, whole heads or part of them)
* norm    - the same with an RMSNorm of every query and key head in front of the rotation
* append  - that pass over a fused QKV row, ending in the paged cache (quantised or plain pages) that decode attention reads
* fork, churn - pages of a cache: sequences forked (shared pages, copied last page), released, reserved, the pool compacted

`run` computes them in elementary torch operations, or, with `own` set, through the framework's entry points.
"""
import math

import torch

own = False      # True: run() calls the framework's operators

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
HEAD_DIM, PAGE, KV_GROUP = 128, 16, 32
THETA, EPS = 500000.0, 1e-6


def listed():
    return [
        # one decoded token of one request with an adapter beside an attention output projection: the smallest call
        dict(name="lora_q4_b1", op="lora", bits=4, rows=1, n=4096, k=4096, group=64, adapters=8, rank=16, run_length=1, dtype="fp16"),
        # a decode batch whose requests use adapters of different ranks (some none) beside a fused QKV projection
        dict(name="lora_q4_b32_mixed_bf16", op="lora", bits=4, rows=32, n=6144, k=4096, group=64, adapters=24, rank=64, run_length=1,
             dtype="bf16"),
        # sizes and a rank that fit no tile
        dict(name="lora_q8_b5_odd", op="lora", bits=8, rows=5, n=5003, k=2592, group=32, adapters=3, rank=12, run_length=1, dtype="fp16"),
        # chunks of four prompts, each with its adapter, through an up projection: the largest product
        dict(name="lora_q4_prompt512", op="lora", bits=4, rows=512, n=14336, k=4096, group=64, adapters=4, rank=64, run_length=128,
             dtype="fp16"),
        # a decode batch far into long contexts, half layout: the smallest rotation
        dict(name="rope_half_b16", op="rope", tokens=16, q_heads=32, kv_heads=8, rotary=128, layout="half", reach=131072, dtype="bf16"),
        # prompts of 8192 tokens, slices of the fused projection's rows, half of each head turned
        dict(name="rope_part_prompt8192", op="rope", tokens=8192, q_heads=32, kv_heads=8, rotary=64, layout="interleaved", reach=8192,
             dtype="fp16"),
        # head norms and rotation of a few decoded tokens, and of an odd number of prompt tokens
        dict(name="norm_half_b4", op="norm", tokens=4, q_heads=32, kv_heads=8, rotary=128, layout="half", reach=8192, dtype="fp16"),
        dict(name="norm_prompt4099_bf16", op="norm", tokens=4099, q_heads=32, kv_heads=8, rotary=128, layout="interleaved", reach=8192,
             dtype="bf16"),
        # a decode step's rows into a quantised cache, with head norms, and read back
        dict(name="append_q8_b32", op="append", kind="q8", tokens=32, sequences=32, q_heads=32, kv_heads=8, rotary=128, layout="half",
             norm=True, dtype="fp16"),
        # prompts of ragged lengths that continue at positions inside a page, into plain bf16 pages
        dict(name="append_bf16_prompt8185", op="append", kind="plain", tokens=8185, sequences=7, q_heads=32, kv_heads=8, rotary=128,
             layout="interleaved", norm=True, dtype="bf16"),
        # four sequences forked into sixteen more (parallel sampling) over the quantised caches of 32 layers
        dict(name="fork_q8_l32", op="fork", kind="q8", layers=32, kv_heads=8, parents=4, children=16, max_len=250),
        # two generations of sequences released, compacted and reserved in turn over the plain caches of 4 layers
        dict(name="churn_bf16_l4", op="churn", kind="plain", layers=4, kv_heads=8, sequences=16, max_len=1024),
    ]


def _log_int(rng, lo, hi, multiple=1):
    """An integer in [lo, hi], spread over the logarithm, rounded down to a multiple."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, v)) // multiple * multiple


def draw(rng):
    op = rng.choice(["lora", "lora", "lora", "rope", "norm", "append", "append", "fork", "churn"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "lora":
        group = rng.choice([32, 64, 64, 128])
        rows = _log_int(rng, 1, 512)
        return dict(op=op, bits=rng.choice([4, 4, 8]), rows=rows, n=_log_int(rng, 1024, 14336), k=_log_int(rng, 1024, 4096, group),
                    group=group, adapters=_log_int(rng, 1, 32), rank=rng.choice([4, 8, 12, 16, 16, 24, 32, 64]),
                    run_length=1 if rows < 64 else rng.choice([1, 37, 128]), dtype=dtype)
    heads = rng.choice([2, 4, 8, 8])
    if op in ("rope", "norm", "append"):
        case = dict(op=op, tokens=_log_int(rng, 1, 8192), q_heads=heads * rng.choice([1, 4, 4, 8]), kv_heads=heads,
                    rotary=rng.choice([128, 128, 64, 32]), layout=rng.choice(["interleaved", "half"]), dtype=dtype)
        if op != "append":
            return dict(case, reach=rng.choice([4096, 8192, 131072]))
        case["tokens"] = _log_int(rng, 1, 8185)
        kind = rng.choice(["q8", "q4", "plain"])
        # 4-bit codes are wide steps: a value on the border of two differs between sums in another order, so these go without norms
        return dict(case, kind=kind, sequences=max(1, case["tokens"] // _log_int(rng, 1, 512)), norm=kind != "q4" and rng.random() < 0.7)
    kind = rng.choice(["q8", "q4", "plain"])
    if op == "fork":
        return dict(op=op, kind=kind, layers=_log_int(rng, 1, 32), kv_heads=heads, parents=_log_int(rng, 1, 6),
                    children=_log_int(rng, 1, 16), max_len=_log_int(rng, 20, 250))
    return dict(op=op, kind=kind, layers=_log_int(rng, 1, 4), kv_heads=heads, sequences=_log_int(rng, 2, 16),
                max_len=_log_int(rng, 20, 1024))


# ---- inputs ---------------------------------------------------------------------------------------------------------
class _Source:
    """Random tensors on the GPU from one seed."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, dtype=torch.float16, std=1.0):
        return (torch.randn(shape, generator=self.gen, device="cuda") * std).to(dtype)

    def ints(self, lo, hi, *shape, dtype=torch.int32):
        return torch.randint(lo, hi, shape, generator=self.gen, device="cuda", dtype=dtype)

    def order(self, n):
        return torch.randperm(n, generator=self.gen, device="cuda")


def _groups(n, size):
    return -(-n // size)


def _spread(count, lo, hi):
    """`count` lengths spread evenly over [lo, hi]: the bytes of a case do not depend on the seed."""
    return [hi] if count == 1 else [lo + (hi - lo) * i // (count - 1) for i in range(count)]


def _ranks(case):
    """Ranks of the adapters: the largest, half and a quarter of it in turn."""
    return [max(1, case["rank"] >> (i % 3)) for i in range(case["adapters"])]


def _adapter_ids(case):
    """Adapter of every row: runs of `run_length` rows take the adapters in turn; of single rows every ninth has none."""
    runs = [(i // case["run_length"]) for i in range(case["rows"])]
    return [-1 if case["run_length"] == 1 and r % 9 == 8 else (5 * r + 1) % case["adapters"] for r in runs]


def _tables(rotary, reach):
    inv = THETA ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    angle = torch.arange(reach, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.cos(angle).float().contiguous(), torch.sin(angle).float().contiguous()


def _append_spans(case):
    """(start, count) of the new tokens of every sequence; starts inside pages."""
    b, t = case["sequences"], case["tokens"]
    counts = [t // b + (1 if i < t % b else 0) for i in range(b)]
    if t > 4 * b:      # ragged: neighbours trade tokens
        for i in range(0, b - 1, 2):
            counts[i], counts[i + 1] = counts[i] - counts[i] // 3, counts[i + 1] + counts[i] // 3
    return [(11 * i % 37, n) for i, n in enumerate(counts)]


def _empty_pool(src, kind, layers, pages, heads, dtype):
    """Pool tensors with leftovers of earlier sequences in them: (codes or values of K, of V, scales of K, of V)."""
    if kind == "plain":
        return [src.normal(layers, pages, PAGE, heads, HEAD_DIM, dtype=dtype) for _ in range(2)]
    width = HEAD_DIM if kind == "q8" else HEAD_DIM // 2
    codes = [src.ints(0, 256, layers, pages, PAGE, heads, width, dtype=torch.uint8) for _ in range(2)]
    if kind == "q8":
        codes = [c.clamp_min_(1) for c in codes]
    scales = [src.normal(layers, pages, PAGE, heads, HEAD_DIM // KV_GROUP, std=0.01).abs_() for _ in range(2)]
    return codes + scales


def prepare(case, seed):
    src = _Source(seed)
    return dict(globals()["_prepare_" + case["op"]](case, src), op=case["op"])


def _prepare_lora(case, src):
    dtype = DTYPES[case["dtype"]]
    n, k, bits, g, count, rank = (case[key] for key in ("n", "k", "bits", "group", "adapters", "rank"))
    top = (1 << bits) - 1
    groups = _groups(k, g)
    # affine codes as a quantiser leaves them: weights of deviation 0.02 over about six deviations
    scales = (0.12 / top * (1 + 0.2 * src.normal(n, groups, dtype=torch.float32))).abs().to(torch.float16)
    zeros = src.ints(top // 2, top // 2 + 2, n, groups).to(torch.float16)
    codes = src.ints(0, 256, n, k * bits // 8, dtype=torch.uint8)
    ranks = torch.tensor(_ranks(case), dtype=torch.int32, device="cuda")
    return dict(x=src.normal(case["rows"], k, dtype=dtype), w=codes, scales=scales, zeros=zeros, bits=bits, group=g,
                a=src.normal(count, rank, k, dtype=dtype, std=k ** -0.5), b=src.normal(count, n, rank, dtype=dtype, std=0.3),
                scaling=(0.5 + torch.rand(count, generator=src.gen, device="cuda")), ranks=ranks,
                ids=torch.tensor(_adapter_ids(case), dtype=torch.int32, device="cuda"))


def _qkv(case, src):
    """(fused rows [T, Hq + 2 Hkv, D], norm weights of the query and key heads)"""
    heads = case["q_heads"] + 2 * case["kv_heads"]
    rows = src.normal(case["tokens"], heads, HEAD_DIM, dtype=DTYPES[case["dtype"]])
    weights = [(1 + 0.1 * src.normal(HEAD_DIM, dtype=torch.float32)).to(rows.dtype) for _ in range(2)]
    return rows, weights


def _prepare_rope(case, src):
    rows, weights = _qkv(case, src)
    hq, hkv = case["q_heads"], case["kv_heads"]
    cos, sin = _tables(case["rotary"], case["reach"])
    return dict(q=rows[:, :hq], k=rows[:, hq:hq + hkv], cos=cos, sin=sin, layout=case["layout"], weights=weights,
                positions=src.ints(0, case["reach"], case["tokens"]))


_prepare_norm = _prepare_rope


def _prepare_append(case, src):
    rows, weights = _qkv(case, src)
    spans = _append_spans(case)
    blocks = [_groups(start + n, PAGE) for start, n in spans]
    pages, width = sum(blocks) + 3, max(blocks)
    order = src.order(pages).to(torch.int32)
    col = torch.arange(width, device="cuda")[None]
    used = col < torch.tensor(blocks, device="cuda")[:, None]
    rank = torch.cumsum(used.reshape(-1), 0).reshape(used.shape) - 1
    table = torch.where(used, order[rank.clamp_min(0)], -1).to(torch.int32).contiguous()
    count = torch.tensor([n for _, n in spans], device="cuda")
    first = torch.cumsum(count, 0) - count
    seq = torch.repeat_interleave(torch.arange(len(spans), device="cuda"), count)
    start = torch.tensor([s for s, _ in spans], device="cuda")
    positions = start[seq] + torch.arange(case["tokens"], device="cuda") - first[seq]
    pool = [t[0] for t in _empty_pool(src, case["kind"], 1, pages, case["kv_heads"], rows.dtype)]
    cos, sin = _tables(case["rotary"], PAGE * width)
    return dict(qkv=rows.reshape(case["tokens"], -1), q_heads=case["q_heads"], weights=weights if case["norm"] else [None, None],
                cos=cos, sin=sin, layout=case["layout"], positions=positions.to(torch.int32), sequences=seq.to(torch.int32), pool=pool,
                kind=case["kind"], table=table, lengths=(start + count).to(torch.int32))


def _refs_of(table, pages):
    used = table[table >= 0].to(torch.int64)
    return torch.bincount(used, minlength=pages).to(torch.int32)


def _fork_sizes(case):
    """(lengths of the parents, pages they hold, blocks of a row, pages of the pool)"""
    lengths = _spread(case["parents"], max(1, case["max_len"] // 3), case["max_len"])
    held = [_groups(n, PAGE) for n in lengths]
    return lengths, held, max(held) + 2, 2 * (sum(held) + case["children"]) + 5


def _prepare_fork(case, src):
    """Parents on shuffled pages; the rows of the children still hold a page each of an earlier sequence."""
    lengths, held, width, pages = _fork_sizes(case)
    parents, children = case["parents"], case["children"]
    order = src.order(pages).to(torch.int32)
    table = torch.full((parents + children, width), -1, dtype=torch.int32, device="cuda")
    used = torch.arange(width, device="cuda")[None] < torch.tensor(held, device="cuda")[:, None]
    table[:parents][used] = order[:sum(held)]
    table[parents:, 0] = order[sum(held):sum(held) + children]
    return dict(pool=_empty_pool(src, case["kind"], case["layers"], pages, case["kv_heads"], torch.bfloat16), kind=case["kind"],
                table=table, refs=_refs_of(table, pages),
                lengths=torch.tensor(lengths + [PAGE] * children, dtype=torch.int32, device="cuda"),
                parents=(torch.arange(children, device="cuda") % parents).to(torch.int32),
                children=(parents + src.order(children)).to(torch.int32))


def _churn_sizes(case):
    """(lengths of the rows, pages they hold, blocks of a row, pages of the pool); the two generations hold one half of the rows each"""
    lengths = _spread(case["sequences"], max(1, case["max_len"] // 2), case["max_len"])
    held = [_groups(n, PAGE) for n in lengths]
    return lengths, held, max(held) + 1, sum(held) + 7


def _prepare_churn(case, src):
    """The even rows hold the low pages, the odd rows the ones behind them, shuffled."""
    lengths, held, width, pages = _churn_sizes(case)
    b = case["sequences"]
    low = sum(held[0::2])
    pages_of = torch.cat([src.order(low), low + src.order(sum(held) - low)]).to(torch.int32)
    used = torch.arange(width, device="cuda")[None] < torch.tensor(held, device="cuda")[:, None]
    turn = torch.cat([torch.arange(0, b, 2, device="cuda"), torch.arange(1, b, 2, device="cuda")])
    rows = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    rows[used[turn]] = pages_of
    table = torch.empty_like(rows)
    table[turn] = rows
    want = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    even = torch.arange(b, device="cuda") % 2 == 0
    return dict(pool=_empty_pool(src, case["kind"], case["layers"], pages, case["kv_heads"], torch.bfloat16), kind=case["kind"],
                table=table, refs=_refs_of(table, pages), lengths=want.clone(), turns=[
                    (torch.nonzero(m).reshape(-1).to(torch.int32), torch.where(m, want, 0).to(torch.int32)) for m in (even, ~even)])


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(state):
    return globals()[("_own_" if own else "_plain_") + state["op"]](state)


# .... in elementary operations
def _weight32(st):
    n, g = st["w"].shape[0], st["group"]
    codes = st["w"]
    if st["bits"] == 4:
        codes = torch.stack((codes & 15, codes >> 4), dim=-1).reshape(n, -1)
    k = codes.shape[1]
    scales, zeros = (t.float().repeat_interleave(g, 1)[:, :k] for t in (st["scales"], st["zeros"]))
    return (codes.float() - zeros) * scales


def _plain_lora(st):
    x, a, b, ids = st["x"].float(), st["a"].float(), st["b"].float(), st["ids"].long()
    count, rank, k = a.shape
    y = x @ _weight32(st).t()
    mine = ids[:, None] == torch.arange(count, device=x.device)
    within = torch.arange(rank, device=x.device)[None] < st["ranks"][:, None]
    t = (x @ a.reshape(count * rank, k).t()).reshape(-1, count, rank)
    t = t * (mine[:, :, None] & within[None]) * st["scaling"][None, :, None]
    y = y + t.reshape(-1, count * rank) @ b.permute(0, 2, 1).reshape(count * rank, -1)
    return y.to(st["x"].dtype)


def _turn(x, cos, sin, layout):
    """x [T, H, D] in 32 or 64 bits, cos / sin [T, 1, rotary / 2]"""
    r = 2 * cos.shape[-1]
    head, rest = x[..., :r], x[..., r:]
    if layout == "half":
        u, v = head[..., :r // 2], head[..., r // 2:]
        turned = torch.cat((u * cos - v * sin, u * sin + v * cos), dim=-1)
    else:
        u, v = head[..., 0::2], head[..., 1::2]
        turned = torch.stack((u * cos - v * sin, u * sin + v * cos), dim=-1).reshape(head.shape)
    return torch.cat((turned, rest), dim=-1)


def _plain_heads(st, x, weight):
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.float()
    at = st["positions"].long()
    return _turn(y, st["cos"][at][:, None], st["sin"][at][:, None], st["layout"]).to(x.dtype)


def _plain_rope(st):
    return _plain_heads(st, st["q"], None), _plain_heads(st, st["k"], None)


def _plain_norm(st):
    return _plain_heads(st, st["q"], st["weights"][0]), _plain_heads(st, st["k"], st["weights"][1])


def _coded(values, bits):
    """(codes, scales) of symmetric groups: the rule of the quantised cache."""
    top, offset = (127.0, 128.0) if bits == 8 else (7.0, 8.0)
    v = values.reshape(*values.shape[:-1], -1, KV_GROUP).float()
    scale = v.abs().amax(-1, keepdim=True).clamp_min(1e-8) / top
    codes = (torch.round(v / scale).clamp(-top, top) + offset).to(torch.uint8).reshape(values.shape)
    if bits == 4:
        codes = codes[..., 0::2] | (codes[..., 1::2] << 4)
    return codes, scale[..., 0].to(torch.float16)


def _values(codes, scales, bits):
    if bits == 4:
        codes = torch.stack((codes & 15, codes >> 4), dim=-1).reshape(*codes.shape[:-1], -1)
    v = codes.float() - (128.0 if bits == 8 else 8.0)
    return (v.reshape(*v.shape[:-1], -1, KV_GROUP) * scales.float().abs()[..., None]).reshape(v.shape).to(torch.float16)


def _split(st):
    t = st["qkv"].shape[0]
    rows = st["qkv"].reshape(t, -1, HEAD_DIM)
    hq = st["q_heads"]
    hkv = (rows.shape[1] - hq) // 2
    return rows[:, :hq], rows[:, hq:hq + hkv], rows[:, hq + hkv:]


def _slots(st):
    at = st["positions"].long()
    return st["table"][st["sequences"].long(), at // PAGE].long(), at % PAGE


def _plain_append(st):
    q, k, v = _split(st)
    q, k = _plain_heads(st, q, st["weights"][0]), _plain_heads(st, k, st["weights"][1])
    page, slot = _slots(st)
    pool = st["pool"]
    if st["kind"] == "plain":
        pool[0][page, slot] = k
        pool[1][page, slot] = v
        return q, pool[0], pool[1]
    bits = 8 if st["kind"] == "q8" else 4
    pool[0][page, slot], pool[2][page, slot] = _coded(k, bits)
    pool[1][page, slot], pool[3][page, slot] = _coded(v, bits)
    return q, _values(pool[0], pool[2], bits), _values(pool[1], pool[3], bits)


def _plain_release(st, rows):
    rows = rows.long()
    held = st["table"][rows]
    st["refs"].index_add_(0, held.clamp_min(0).reshape(-1).long(), -(held >= 0).to(torch.int32).reshape(-1))
    st["table"][rows] = -1
    st["lengths"][rows] = 0


def _free_pages(refs):
    """Page numbers, the free ones first, in ascending order."""
    return torch.argsort((refs > 0).to(torch.int32), stable=True)


def _plain_fork_rows(st, parents, children):
    parents, children = parents.long(), children.long()
    length = st["lengths"][parents]
    full, rest = length // PAGE, length % PAGE
    col = torch.arange(st["table"].shape[1], device=length.device)[None]
    rows = st["table"][parents]
    shared = (col < full[:, None]) & (rows >= 0)
    part = (col == full[:, None]) & (rest > 0)[:, None] & (rows >= 0)
    st["refs"].index_add_(0, rows.clamp_min(0).reshape(-1).long(), shared.to(torch.int32).reshape(-1))
    rank = torch.cumsum(part.reshape(-1), 0).reshape(part.shape) - 1
    fresh = _free_pages(st["refs"])[rank.clamp_min(0)].to(torch.int32)
    st["table"][children] = torch.where(shared, rows, torch.where(part, fresh, -1))
    st["lengths"][children] = length
    src, dst = rows[part].long(), fresh[part].long()
    st["refs"][dst] = 1
    keep = (torch.arange(PAGE, device=length.device)[None] < rest[part.any(1), None])[None, :, :, None, None]
    for t in st["pool"]:
        t[:, dst] = torch.where(keep, t[:, src], t[:, dst])


def _paged_state(st):
    return list(st["pool"]) + [st["table"], st["lengths"], st["refs"]]


def _plain_fork(st):
    _plain_release(st, st["children"])
    _plain_fork_rows(st, st["parents"], st["children"])
    return _paged_state(st)


def _plain_compact(st):
    refs = st["refs"]
    live = refs > 0
    count = live.sum()
    page = torch.arange(refs.numel(), device=refs.device)
    src, dst = page[live & (page >= count)], page[~live & (page < count)]
    place = page.clone()
    place[src] = dst
    for t in st["pool"]:
        t[:, dst] = t[:, src]
    refs[dst] = refs[src]
    refs[src] = 0
    st["table"].copy_(torch.where(st["table"] >= 0, place[st["table"].clamp_min(0).long()].to(torch.int32), st["table"]))


def _plain_reserve(st, new_tokens):
    lengths = st["lengths"]
    col = torch.arange(st["table"].shape[1], device=lengths.device)[None]
    first, last = lengths // PAGE, (lengths + new_tokens + PAGE - 1) // PAGE
    need = (col >= first[:, None]) & (col < last[:, None]) & (st["table"] < 0)
    rank = torch.cumsum(need.reshape(-1), 0).reshape(need.shape) - 1
    fresh = _free_pages(st["refs"])[rank.clamp_min(0)].to(torch.int32)
    st["refs"][fresh[need].long()] = 1
    st["table"].copy_(torch.where(need, fresh, st["table"]))


def _plain_churn(st):
    for rows, tokens in st["turns"]:
        _plain_release(st, rows)
        _plain_compact(st)
        _plain_reserve(st, tokens)
        st["lengths"] += tokens
    return _paged_state(st)


# .... through the framework's entry points
_modules = {}


def _op(name):
    if name not in _modules:
        import importlib

        import __graft_entry__
        __graft_entry__.load_package()
        _modules[name] = importlib.import_module("mlx_metal_kernels_b200.ops." + name)
    return _modules[name]


def _kept(st, make):
    """What a program keeps between its calls beside the tensors: made on the first pass."""
    if "kept" not in st:
        st["kept"] = make(st)
    return st["kept"]


def _own_lora(st):
    lora = _op("lora_ops")
    adapters = _kept(st, lambda s: lora.LoraAdapters(s["a"], s["b"], s["scaling"], ranks=s["ranks"]))
    return lora.lora_quantized_linear(st["x"], st["w"], st["scales"], st["zeros"], adapters, st["ids"], bits=st["bits"],
                                      group_size=st["group"])


def _own_rope(st):
    return _op("rope_ops").apply_rope(st["q"], st["k"], st["cos"], st["sin"], st["positions"], layout=st["layout"])


def _own_norm(st):
    return _op("rope_ops").head_norm_rope(st["q"], st["k"], *st["weights"], st["cos"], st["sin"], st["positions"], eps=EPS,
                                          layout=st["layout"])


def _cache_of(st, pool):
    kind = _op("paged_quantized_kv_ops").PagedQuantizedKVCache
    return kind(k_pages_q=pool[0], v_pages_q=pool[1], k_scales=pool[2], v_scales=pool[3], block_table=st["table"], lengths=st["lengths"],
                bits=8 if st["kind"] == "q8" else 4, page_size=PAGE, group_size=KV_GROUP,
                original_page_shape=(*pool[0].shape[:3], HEAD_DIM))


def _own_append(st):
    more = dict(sequences=st["sequences"], q_weight=st["weights"][0], k_weight=st["weights"][1], eps=EPS, layout=st["layout"])
    pool = st["pool"]
    if st["kind"] == "plain":
        q = _op("paged_kv_ops").norm_rope_kv_append_pages(st["qkv"], st["cos"], st["sin"], st["positions"], pool[0], pool[1], st["table"],
                                                          st["q_heads"], **more)
        return q, pool[0], pool[1]
    cache = _kept(st, lambda s: _cache_of(s, s["pool"]))
    q = _op("decode_layer_ops").norm_rope_kv_append(st["qkv"], st["cos"], st["sin"], st["positions"], cache, st["q_heads"], **more)
    k, v = _op("paged_quantized_kv_ops").dequantize_kv_pages(cache)
    return q, k, v


def _page_handles(st):
    pages = _op("kv_page_ops")
    layers = list(zip(*st["pool"]))
    caches = layers if st["kind"] == "plain" else [_cache_of(st, layer) for layer in layers]
    return caches, pages.PagePool(st["refs"], page_size=PAGE)


def _own_fork(st):
    pages = _op("kv_page_ops")
    caches, pool = _kept(st, _page_handles)
    pages.release_sequences(pool, st["table"], st["lengths"], st["children"])
    pages.fork_sequences(caches, pool, st["table"], st["lengths"], st["parents"], st["children"])
    return _paged_state(st)


def _own_churn(st):
    pages = _op("kv_page_ops")
    caches, pool = _kept(st, _page_handles)
    for rows, tokens in st["turns"]:
        pages.release_sequences(pool, st["table"], st["lengths"], rows)
        pages.compact_pages(caches, pool, st["table"])
        pages.reserve_pages(pool, st["table"], st["lengths"], tokens)
        st["lengths"] += tokens
    return _paged_state(st)


# ---- from the definition, in 64 bits --------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] in ("fork", "churn"):
        return None      # pages are moved, not computed
    return globals()["_exact_" + case["op"]](prepare(case, seed))


def _exact_lora(st):
    x = st["x"].double()
    n, k = st["w"].shape[0], x.shape[1]
    column = torch.arange(k, device="cuda")
    if st["bits"] == 4:
        q = (st["w"][:, column // 2].long() >> (4 * (column % 2))) & 15
    else:
        q = st["w"].long()
    g = column // st["group"]
    y = torch.einsum("tk,nk->tn", x, (q - st["zeros"].double()[:, g]) * st["scales"].double()[:, g])
    rows = torch.nonzero(st["ids"] >= 0).reshape(-1)
    ids = st["ids"][rows].long()
    low = torch.bmm(st["a"][ids].double(), x[rows, :, None])[..., 0]
    low[torch.arange(low.shape[1], device="cuda")[None] >= st["ranks"][ids, None]] = 0
    y[rows] += st["scaling"].double()[ids, None] * torch.bmm(st["b"][ids].double(), low[..., None])[..., 0]
    return y


def _exact_heads(st, x, weight):
    y = x.double().clone()
    if weight is not None:
        y /= torch.sqrt(torch.linalg.vector_norm(y, dim=-1, keepdim=True) ** 2 / HEAD_DIM + EPS)
        y *= weight.double()
    at = st["positions"].long()
    angle = torch.complex(st["cos"].double()[at], st["sin"].double()[at])[:, None]
    pairs = angle.shape[-1]
    even = torch.arange(pairs, device="cuda") * (1 if st["layout"] == "half" else 2)
    odd = even + (pairs if st["layout"] == "half" else 1)
    z = torch.complex(y[..., even], y[..., odd]) * angle
    y[..., even], y[..., odd] = z.real, z.imag
    return y


def _exact_rope(st):
    return _exact_heads(st, st["q"], None), _exact_heads(st, st["k"], None)


def _exact_norm(st):
    return _exact_heads(st, st["q"], st["weights"][0]), _exact_heads(st, st["k"], st["weights"][1])


def _exact_append(st):
    """A quantised cache holds the rows as the activations' type has them, each value at the nearest step of its group's largest
    magnitude over 127.  4-bit steps are so wide that the borders between them, which the rule draws in 32 bits, decide how
    far a value is off: they have no value in 64 bits."""
    q, k, v = _split(st)
    out = [_exact_heads(st, q, st["weights"][0])]
    page, slot = _slots(st)
    for i, rows in enumerate((_exact_heads(st, k, st["weights"][1]), v.double())):
        if st["kind"] == "q4":
            out.append(None)
            continue
        if st["kind"] == "plain":
            held = st["pool"][i].double()
        else:
            held = _values(st["pool"][i], st["pool"][2 + i], 8).double()
            groups = rows.to(v.dtype).double().unflatten(-1, (-1, KV_GROUP))
            step = groups.abs().amax(-1, keepdim=True).clamp_min(1e-8) / 127
            rows = ((groups / step).round() * step).flatten(-2)
        held[page, slot] = rows
        out.append(held)
    return tuple(out)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def _page_bytes(case):
    """Bytes of one page in all layers."""
    row = {"plain": 2 * HEAD_DIM, "q8": HEAD_DIM + 2 * HEAD_DIM // KV_GROUP, "q4": HEAD_DIM // 2 + 2 * HEAD_DIM // KV_GROUP}[case["kind"]]
    return case["layers"] * 2 * PAGE * case["kv_heads"] * row


def work(case):
    op = case["op"]
    if op == "lora":
        rows, n, k = case["rows"], case["n"], case["k"]
        ranks, ids = _ranks(case), _adapter_ids(case)
        base = n * k * case["bits"] // 8 + 4 * n * _groups(k, case["group"])
        used = sum(ranks[i] for i in set(ids) if i >= 0)
        turned = sum(ranks[i] for i in ids if i >= 0)
        return {"bytes": base + 2 * used * (n + k) + 2 * rows * (n + k), "flops": 2 * rows * n * k + 2 * turned * (n + k)}
    if op in ("rope", "norm", "append"):
        t, hq, hkv = case["tokens"], case["q_heads"], case["kv_heads"]
        values = t * (hq + hkv) * HEAD_DIM
        table = 4 * min(t, case.get("reach", t)) * case["rotary"] + 4 * t
        flops = 3 * t * (hq + hkv) * case["rotary"] + (4 * values if op == "norm" or case.get("norm") else 0)
        if op != "append":
            return {"bytes": 4 * values + table, "flops": flops}
        # the fused rows in, the queries out, one row per token and head into the cache; quantised pages are read back whole
        row = _page_bytes(dict(case, layers=1)) // PAGE
        read_back = 0
        if case["kind"] != "plain":
            pages = sum(_groups(s + n, PAGE) for s, n in _append_spans(case)) + 3
            read_back = pages * (_page_bytes(dict(case, layers=1)) + 4 * PAGE * hkv * HEAD_DIM)
        return {"bytes": 2 * t * (hq + 2 * hkv) * HEAD_DIM + 2 * t * hq * HEAD_DIM + t * row + table + 8 * t + read_back, "flops": flops}
    if op == "fork":
        lengths, _, width, pages = _fork_sizes(case)
        slots = sum(lengths[i % case["parents"]] % PAGE for i in range(case["children"]))
        index = 4 * (2 * case["children"] * width + pages)
        return {"bytes": 2 * slots * _page_bytes(case) // PAGE + index, "flops": 0}
    lengths, held, width, pages = _churn_sizes(case)
    moved = 2 * min(sum(held[0::2]), sum(held[1::2]))
    return {"bytes": 2 * moved * _page_bytes(case) + 4 * 4 * (pages + case["sequences"] * width), "flops": 0}
