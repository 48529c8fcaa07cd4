"""GPU page operators against a plain sequential restatement on the host: tables, counts, lengths and every byte of every layer."""
import importlib
import random

import pytest
import torch

import __graft_entry__ as entry
from helpers import cabi, gen, pq_ops

pytestmark = pytest.mark.gpu
entry.load_package()
pages = importlib.import_module("mlx_metal_kernels_b200.ops.kv_page_ops")


# ---- the rules, one step after another ------------------------------------------------------------------------------
class Model:
    """Tables, counts, lengths and tensors [pages, P, ...] on the host; a call that cannot be served leaves them alone."""

    def __init__(self, table, refs, lengths, tensors, P):
        self.table, self.refs, self.lengths, self.tensors, self.P = table.clone(), refs.clone(), lengths.clone(), [t.clone() for t in tensors], P
        self.width = table.shape[1]

    def free(self):
        return [i for i, r in enumerate(self.refs.tolist()) if r <= 0]

    def reserve(self, new):
        need = []
        for b, n in enumerate(new):
            length = int(self.lengths[b])
            if n and -(-(length + n) // self.P) > self.width:
                return 8
            if n:
                need += [(b, j) for j in range(length // self.P, -(-(length + n) // self.P)) if self.table[b, j] < 0]
        free = self.free()
        if len(free) < len(need):
            return 9
        for (b, j), page in zip(need, free):
            self.table[b, j], self.refs[page] = page, 1
        return 0

    def release(self, rows):
        event = 0
        for b in rows:
            if b < 0:
                continue
            if b >= len(self.table):
                event = 8
                continue
            for j in range(self.width):
                page = int(self.table[b, j])
                if page >= 0:
                    if page >= len(self.refs) or self.refs[page] <= 0:
                        event = 8
                    else:
                        self.refs[page] -= 1
                self.table[b, j] = -1
            self.lengths[b] = 0
        return event

    def copy(self, src, dst):
        pairs = [(s, d) for s, d in zip(src, dst) if s >= 0 and d >= 0]
        n = len(self.refs)
        dsts = [d for _, d in pairs]
        if any(s >= n or d >= n for s, d in pairs) or len(set(dsts)) < len(dsts) or set(dsts) & {s for s, _ in pairs}:
            return 8
        for s, d in pairs:
            for t in self.tensors:
                t[d] = t[s]
        return 0

    def fork(self, parents, children):
        pairs = [(p, c) for p, c in zip(parents, children) if p >= 0 and c >= 0]
        kids = [c for _, c in pairs]
        B = len(self.table)
        if any(p >= B or c >= B for p, c in pairs) or len(set(kids)) < len(kids) or set(kids) & {p for p, _ in pairs}:
            return 8
        for p, c in pairs:
            if not 0 <= self.lengths[p] <= self.width * self.P or self.lengths[c] != 0 or bool((self.table[c] >= 0).any()):
                return 8
        part = [(p, c) for p, c in pairs if self.lengths[p] % self.P and self.table[p, self.lengths[p] // self.P] >= 0]
        free = self.free()
        if len(free) < len(part):
            return 9
        for (p, c), page in zip(part, free):
            j, rest = int(self.lengths[p]) // self.P, int(self.lengths[p]) % self.P
            self.table[c, j], self.refs[page] = page, 1
            for t in self.tensors:
                t[page, :rest] = t[int(self.table[p, j]), :rest]
        for p, c in pairs:
            for j in range(int(self.lengths[p]) // self.P):
                page = int(self.table[p, j])
                if page >= 0:
                    self.table[c, j] = page
                    self.refs[page] += 1
            self.lengths[c] = self.lengths[p]
        return 0

    def compact(self):
        live = [i for i, r in enumerate(self.refs.tolist()) if r > 0]
        low = set(live)
        holes = [i for i in range(len(live)) if i not in low]
        remap = {i: i for i in live}
        for src, dst in zip([i for i in live if i >= len(live)], holes):
            remap[src] = dst
            for t in self.tensors:
                t[dst] = t[src]
            self.refs[dst], self.refs[src] = int(self.refs[src]), 0
        for b in range(len(self.table)):
            for j in range(self.width):
                page = int(self.table[b, j])
                self.table[b, j] = remap.get(page, page) if page >= 0 else page
        return [remap.get(i, -1) for i in range(len(self.refs))]


KINDS = {  # dtype and widths of the last axis (values, scales); heads
    "q8": (torch.uint8, 128, 4, 8), "q4": (torch.uint8, 64, 4, 2), "plain": (torch.bfloat16, 128, 0, 4), "words": (torch.float16, 2, 0, 3),
    "bytes": (torch.uint8, 5, 1, 3),
}


class World:
    """A pool on the GPU with its caches, and the same on the host."""

    def __init__(self, cuda, kind, layers, num_pages, P, B, width, seed):
        g = gen(seed)
        dtype, d, ds, heads = KINDS[kind]
        self.host = []
        for _ in range(layers):
            values = [torch.randint(0, 256, (num_pages, P, heads, d * (1 if dtype == torch.uint8 else 2)), generator=g, dtype=torch.int32)
                      .to(torch.uint8).view(dtype) for _ in range(2)]
            self.host.append(values + [torch.randn((num_pages, P, heads, ds), generator=g).to(torch.float16) for _ in range(2 if ds else 0)])
        dev = [[t.to(cuda) for t in layer] for layer in self.host]
        self.flat = [t for layer in dev for t in layer]
        if ds:
            self.caches = [pq_ops.PagedQuantizedKVCache(*layer, None, None, bits=8, page_size=P) for layer in dev]
        else:
            self.caches = [tuple(layer) for layer in dev]
        self.table = torch.full((B, width), -1, dtype=torch.int32, device=cuda)
        self.lengths = torch.zeros(B, dtype=torch.int32, device=cuda)
        self.pool = pages.PagePool.empty(num_pages, P, cuda)
        self.model = Model(self.table.cpu(), self.pool.ref_counts.cpu(), self.lengths.cpu(), [t.view(torch.uint8) for layer in self.host for t in layer], P)
        cabi.device_status()

    def check(self, event):
        assert cabi.device_status() == event
        m = self.model
        assert torch.equal(self.table.cpu(), m.table) and torch.equal(self.lengths.cpu(), m.lengths)
        assert torch.equal(self.pool.ref_counts.cpu(), m.refs)
        for a, b in zip(self.flat, m.tensors):
            assert torch.equal(a.cpu().view(torch.uint8), b)

    def ints(self, v):
        return torch.tensor(v, dtype=torch.int32, device=self.table.device)

    def grow(self, new):
        """Reserves and lengthens on both sides."""
        if isinstance(new, int):
            pages.reserve_pages(self.pool, self.table, self.lengths, new)
            new = [new] * len(self.model.table)
        else:
            pages.reserve_pages(self.pool, self.table, self.lengths, self.ints(new))
        event = self.model.reserve(new)
        self.check(event)
        if event == 0:
            self.lengths += self.ints(new)
            self.model.lengths += torch.tensor(new, dtype=torch.int32)
        return event

    def release(self, rows):
        pages.release_sequences(self.pool, self.table, self.lengths, self.ints(rows))
        self.check(self.model.release(rows))

    def fork(self, parents, children):
        pages.fork_sequences(self.caches, self.pool, self.table, self.lengths, self.ints(parents), self.ints(children))
        event = self.model.fork(parents, children)
        self.check(event)
        return event

    def copy(self, src, dst):
        pages.copy_pages(self.caches, self.ints(src), self.ints(dst))
        event = self.model.copy(src, dst)
        self.check(event)
        return event

    def compact(self):
        remap = pages.compact_pages(self.caches, self.pool, self.table)
        assert remap.tolist() == self.model.compact()
        self.check(0)


@pytest.mark.parametrize("kind,layers,P", [("q8", 2, 16), ("q4", 3, 16), ("plain", 1, 16), ("words", 2, 5), ("bytes", 2, 3), ("plain", 2, 1)])
def test_a_life_of_sequences(cuda, kind, layers, P):
    w = World(cuda, kind, layers, 60, P, 9, 12, seed=layers + P)
    assert w.grow([3 * P, P + 1, 1, 0, 0, 2 * P - 1, 0, 0, 0]) == 0
    assert w.grow(1) == 0                                                # the full pages of row 0 are followed by a new one
    w.release([3, 4, 6, 7, 8])
    assert w.fork([0, 0, 1, 2], [3, 4, 7, 8]) == 0
    assert w.fork([5], [6]) == 0
    w.release([0, 5])                                                    # shared pages stay with the children
    assert w.grow([0, P, 0, 2 * P, 1, 0, 0, 3, 0]) == 0
    w.compact()
    w.compact()                                                          # nothing left to move
    assert w.fork([3], [0]) == 0
    w.release([1, 3, 0, 4, 4, -1])
    w.compact()
    w.release(list(range(9)))
    assert w.pool.ref_counts.sum() == 0
    w.compact()


@pytest.mark.parametrize("seed", range(4))
def test_random_lives(cuda, seed):
    rng = random.Random(seed)
    P, B = rng.choice([1, 4, 16]), 24
    w = World(cuda, rng.choice(["q8", "q4", "plain"]), rng.choice([1, 2]), rng.choice([70, 200]), P, B, 9, seed)
    seen = set()
    for _ in range(25):
        empty = [b for b in range(B) if w.model.lengths[b] == 0 and not (w.model.table[b] >= 0).any()]
        held = [b for b in range(B) if w.model.lengths[b] > 0]
        step = rng.choice(["grow", "grow", "fork", "fork", "release", "compact", "copy"])
        if step == "grow":
            seen.add(w.grow([rng.choice([0, 0, 1, P, 2 * P + 1]) for _ in range(B)]))
        elif step == "fork" and held and empty:
            kids = rng.sample(empty, rng.randint(1, min(len(empty), 6))) + ([-1] if rng.random() < 0.3 else [])
            seen.add(w.fork([rng.choice(held) for _ in kids], kids))
        elif step == "release":
            w.release([rng.randrange(-1, B) for _ in range(rng.randint(1, 8))])
        elif step == "compact":
            w.compact()
        elif step == "copy":
            n = rng.randint(1, 20)
            picked = rng.sample(range(len(w.model.refs)), 2 * n)
            w.copy(picked[:n] + [0], picked[n:] + [-1])
    assert 0 in seen


def test_refused_calls_change_nothing(cuda):
    w = World(cuda, "q8", 2, 12, 16, 6, 4, seed=1)
    assert w.grow([40, 16, 1, 0, 0, 0]) == 0                             # 3 + 1 + 1 pages
    assert w.grow([0, 50, 0, 0, 0, 0]) == 8                              # past the end of a table row
    assert w.grow([0, 0, 0, 64, 64, 0]) == 9                             # 8 pages of 7
    assert w.grow([24, 0, 0, 0, 0, 0]) == 0                              # to the last slot of the row
    assert w.grow([1, 0, 0, 0, 0, 0]) == 8
    for parents, children in (([0, 1], [3, 3]), ([0, 3], [3, 4]), ([0], [0]), ([6], [3]), ([0], [6]), ([0], [1]), ([2 ** 30], [5])):
        assert w.fork(parents, children) == 8
    pages.reserve_pages(w.pool, w.table, w.lengths, w.ints([0, 0, 0, 5, 0, 0]))
    assert w.model.reserve([0, 0, 0, 5, 0, 0]) == 0
    assert w.fork([0], [3]) == 8                                         # empty, but it holds a reserved page
    w.release([3])
    assert w.fork([0, 1, -1, 2], [3, 4, 5, -1]) == 0
    assert w.grow([0, 0, 0, 0, 0, 64]) == 0
    assert w.fork([2], [5]) == 8
    w.release([1])
    assert w.grow([0, 8, 0, 0, 0, 0]) == 0
    w.release([5])
    while w.model.free()[1:]:
        w.model.refs[w.model.free()[0]] = 1
    w.pool.ref_counts.copy_(w.model.refs)
    w.release([4])
    while w.model.free():
        w.model.refs[w.model.free()[0]] = 1
    w.pool.ref_counts.copy_(w.model.refs)
    assert w.fork([2], [4]) == 9                                         # no free page for the copy
    for src, dst in (([0, 1], [5, 5]), ([0, 5], [5, 6]), ([3], [3]), ([12], [0]), ([0], [12]), ([2, 2 ** 30], [3, 4])):
        assert w.copy(src, dst) == 8
    assert w.copy([0, 0, -5, 1], [5, 6, 7, -1]) == 0                     # one source twice; padding
    w.release([6])                                                       # a row that does not exist
    w.release([-1, -2])


def test_inconsistent_counts_are_reported(cuda):
    w = World(cuda, "words", 1, 6, 4, 3, 2, seed=2)
    assert w.grow([8, 4, 0]) == 0
    w.table[1, 1] = w.model.table[1, 1] = 5                              # free, but named
    w.release([1])                                                       # (the check inside expects event 8)
    w.table[2, 0] = w.model.table[2, 0] = 77                             # no page of the pool
    w.release([2])


def test_empty_calls(cuda):
    w = World(cuda, "plain", 1, 6, 4, 3, 2, seed=3)
    none = w.ints([])
    pages.release_sequences(w.pool, w.table, w.lengths, none)
    pages.copy_pages(w.caches, none, none)
    pages.fork_sequences(w.caches, w.pool, w.table, w.lengths, none, none)
    assert w.grow(0) == 0
    w.compact()
    assert w.fork([0, 1], [1, 2]) == 8
    assert w.fork([0, 0], [1, 2]) == 0                                   # of an empty sequence: empty ones


def test_many_layers(cuda):
    """More tensors than one launch names."""
    w = World(cuda, "words", 150, 10, 4, 4, 3, seed=4)
    assert w.grow([7, 3, 0, 0]) == 0
    assert w.fork([0, 1], [2, 3]) == 0
    w.release([0])
    w.compact()
    assert w.copy([0, 1], [8, 9]) == 0


def test_large_pools(cuda):
    """Tens of thousands of pages: every warp of the plans has more than one piece."""
    w = World(cuda, "bytes", 1, 40000, 1, 300, 200, seed=5)
    rng = random.Random(5)
    assert w.grow([rng.randint(0, 200) for _ in range(300)]) == 0
    w.release(list(range(0, 300, 2)))
    empty = [b for b in range(300) if w.model.lengths[b] == 0]
    held = [b for b in range(300) if w.model.lengths[b] > 0]
    assert w.fork([rng.choice(held) for _ in empty], empty) == 0
    w.release(held[::3])
    w.compact()


def test_long_lists(cuda):
    """More sequences, children and pages in a call than the plans have threads, and padding in between."""
    B = 2600
    w = World(cuda, "bytes", 1, 4500, 3, B, 4, seed=8)
    assert w.grow([4] * 1300 + [0] * 1300) == 0
    children = [-1 if i % 7 == 0 else 1300 + i for i in range(1300)]
    assert w.fork(list(range(1300)), children) == 0
    assert w.copy(list(range(1500)), list(range(2999, 1499, -1))) == 0
    assert w.copy(list(range(1500)), list(range(2998, 1498, -1))) == 8
    w.release([b for b in range(B) if b % 3] * 2)
    w.compact()


def test_offsets_past_32_bits(cuda):
    """Pages behind the first 4 GB of a tensor."""
    n, shape = 280000, (16, 8, 128)
    K = torch.empty((n, *shape), dtype=torch.uint8, device=cuda)
    V = torch.empty_like(K)
    scales = torch.empty((n, 16, 8, 4), dtype=torch.float16, device=cuda)
    g = gen(6)
    for t in (K, V):
        t[-3:].copy_(torch.randint(0, 256, (3, *shape), generator=g, dtype=torch.int32))
    scales[-3:] = 2.0
    cache = pq_ops.PagedQuantizedKVCache(K, V, scales, scales, None, None)
    table = torch.tensor([[n - 1, n - 3, -1]], dtype=torch.int32, device=cuda)
    want = [t[[n - 1, n - 3]].clone() for t in (K, V, scales)]
    pool = pages.PagePool.from_block_table(table, n)
    pages.copy_pages(cache, torch.tensor([n - 1], dtype=torch.int32, device=cuda), torch.tensor([n - 2], dtype=torch.int32, device=cuda))
    assert torch.equal(K[n - 2], want[0][0])
    pages.compact_pages(cache, pool, table)
    assert table.tolist() == [[1, 0, -1]] and pool.ref_counts[:3].tolist() == [1, 1, 0]
    assert all(torch.equal(t[[1, 0]], x) for t, x in zip((K, V, scales), want))
    assert cabi.device_status() == 0


def test_captured_calls(cuda):
    """A captured round of release, fork, reserve and compact, replayed over changed indices, and on a stream of its own."""
    a, b = (World(cuda, "q8", 2, 40, 16, 6, 6, seed=7) for _ in range(2))
    for w in (a, b):
        assert w.grow([40, 33, 0, 0, 16, 0]) == 0
    parents, children, gone, more = b.ints([0, 1, -1]), b.ints([2, 3, 5]), b.ints([4, -1]), b.ints([0, 1, 2, 3, 40, 0])

    def round_():
        pages.release_sequences(b.pool, b.table, b.lengths, gone)
        pages.fork_sequences(b.caches, b.pool, b.table, b.lengths, parents, children)
        pages.reserve_pages(b.pool, b.table, b.lengths, more)
        b.lengths += more
        return pages.compact_pages(b.caches, b.pool, b.table)

    def same(p, c, g, m):
        a.release(g)
        assert a.fork(p, c) == 0
        assert a.grow(m) == 0
        a.compact()
        b.model = a.model
        b.check(0)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        round_()
    graph.replay()
    same([0, 1, -1], [2, 3, 5], [4, -1], [0, 1, 2, 3, 40, 0])
    for t, v in ((parents, [3, 4, 2]), (children, [0, -1, 5]), (gone, [0, 0]), (more, [1, 0, 0, 0, 0, 20])):
        t.copy_(torch.tensor(v))
    graph.replay()
    same([3, 4, 2], [0, -1, 5], [0, 0], [1, 0, 0, 0, 0, 20])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for t, v in ((parents, [1, -1, -1]), (children, [4, 0, 0]), (gone, [4, 5]), (more, [0, 0, 1, 0, 0, 0])):
        t.copy_(torch.tensor(v))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        round_()
    side.synchronize()
    same([1, -1, -1], [4, 0, 0], [4, 5], [0, 0, 1, 0, 0, 0])
