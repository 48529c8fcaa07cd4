"""Refusals of the page operators (CPU only; what is checked on the device is tested in test_gpu_kv_pages.py)."""
import ctypes
import importlib
from types import SimpleNamespace

import pytest
import torch

import __graft_entry__ as entry
from helpers import cabi, pq_ops

entry.load_package()
pages = importlib.import_module("mlx_metal_kernels_b200.ops.kv_page_ops")
i32 = lambda *v: torch.tensor(v, dtype=torch.int32)


def setup(num_pages=8, P=4, B=3, max_blocks=2):
    pool = pages.PagePool.empty(num_pages, P)
    return pool, torch.full((B, max_blocks), -1, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)


def plain(num_pages=8, P=4, Hkv=2, D=8, dtype=torch.float16):
    return torch.zeros(num_pages, P, Hkv, D, dtype=dtype), torch.zeros(num_pages, P, Hkv, D, dtype=dtype)


def quantised(num_pages=8, P=4):
    z = lambda d, t: torch.zeros(num_pages, P, 2, d, dtype=t)
    return pq_ops.PagedQuantizedKVCache(z(8, torch.uint8), z(8, torch.uint8), z(1, torch.float16), z(1, torch.float16), None, None,
                                        page_size=P, original_page_shape=(num_pages, P, 2, 8))


def test_pools():
    table = i32(0, 3, 3, -1).reshape(2, 2)
    pool = pages.PagePool.from_block_table(table, 5)
    assert pool.ref_counts.tolist() == [1, 0, 0, 2, 0] and pool.num_pages == 5
    with pytest.raises(ValueError, match="outside a pool"):
        pages.PagePool.from_block_table(table, 3)
    with pytest.raises(ValueError, match="num_pages"):
        pages.PagePool.empty(0)
    for bad in (torch.zeros(0, dtype=torch.int32), torch.zeros(3), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(6, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="ref_counts"):
            pages.PagePool(bad).validate()
    with pytest.raises(ValueError, match="page_size"):
        pages.PagePool(torch.zeros(3, dtype=torch.int32), 0).validate()


def test_tables_and_indices():
    pool, table, lengths = setup()
    for bad in (table.long(), table[:, ::2], table[0], table[:0]):
        with pytest.raises(ValueError, match="block_table"):
            pages.reserve_pages(pool, bad, lengths, 1)
    for bad in (lengths.long(), lengths[:2], torch.zeros(6, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="lengths"):
            pages.release_sequences(pool, table, bad, i32(0))
    for bad in (-1, 2 ** 31):
        with pytest.raises(ValueError, match="new_tokens"):
            pages.reserve_pages(pool, table, lengths, bad)
    with pytest.raises(ValueError, match="new_tokens"):
        pages.reserve_pages(pool, table, lengths, i32(1, 1))
    with pytest.raises(ValueError, match="rows must be"):
        pages.release_sequences(pool, table, lengths, torch.tensor([0]))
    with pytest.raises(ValueError, match="parents and children"):
        pages.fork_sequences([plain()], pool, table, lengths, i32(0), i32(1, 2))
    with pytest.raises(ValueError, match="src_pages and dst_pages"):
        pages.copy_pages([plain()], i32(0), i32(1, 2))
    for call in (lambda: pages.reserve_pages(pool, table, lengths, 1), lambda: pages.release_sequences(pool, table, lengths, i32(0)),
                 lambda: pages.copy_pages(plain(), i32(0), i32(1)), lambda: pages.copy_pages(quantised(), i32(0), i32(1)),
                 lambda: pages.fork_sequences([plain()], pool, table, lengths, i32(0), i32(1)),
                 lambda: pages.compact_pages([quantised()], pool, table)):
        with pytest.raises(cabi.B200QError, match="no CPU route"):
            call()


def test_caches():
    pool, table, lengths = setup()
    for bad, match in (([], "at least one"), ([plain(), plain(D=16)], "one shape"), ([plain(), plain(dtype=torch.bfloat16)], "one shape"),
                       ([plain(), quantised()], "all quantized or all plain"), ([plain(num_pages=9)], "do not fit"), ([plain(P=8)], "do not fit"),
                       ([(plain()[0],) * 3], "pairs"), ([tuple(t.transpose(1, 2) for t in plain())], "contiguous"),
                       ([tuple(t[0] for t in plain())], "contiguous")):
        with pytest.raises(ValueError, match=match):
            pages.compact_pages(bad, pool, table)
    broken = quantised()
    broken.k_scales = broken.v_scales = torch.zeros(7, 4, 2, 1, dtype=torch.float16)
    with pytest.raises(ValueError, match="agree"):
        pages.compact_pages(broken, pool, table)
    broken = quantised()
    broken.k_zeros = broken.k_scales
    with pytest.raises(NotImplementedError):
        pages.compact_pages(broken, pool, table)
    stack = SimpleNamespace(k_codes=torch.zeros(8, 4, 2, 8, dtype=torch.uint8), v_codes=torch.zeros(8, 4, 2, 8, dtype=torch.uint8),
                            k_scales=torch.zeros(8, 4, 2, 1), v_scales=torch.zeros(8, 4, 2, 1))
    groups, shape = pages._cache_tensors([stack, stack], 8, 4)
    assert [len(g) for g in groups] == [4, 4] and shape == (8, 4)
    assert pages._group_args(groups[0])[1:] == (4, 16) and pages._group_args(groups[1])[1:] == (4, 8)


def test_c_abi_refuses_bad_arguments():
    lib = cabi.load()
    one = (ctypes.c_void_p * 2)(16, 16)
    null = (ctypes.c_void_p * 2)(16, None)
    assert lib.b200q_reserve_pages_workspace_bytes(0, 5) == 0 and lib.b200q_compact_pages_workspace_bytes(0) == 0
    assert lib.b200q_reserve_pages_workspace_bytes(3, 8) >= 4 * (2 * 8 + 3)
    cases = {
        "b200q_reserve_pages": ([16, 8, 16, 16, None, 1, 3, 2, 4, 16, 1 << 20, None], ((0, None), (2, None), (3, None), (1, 0), (5, -1), (6, 0),
                                (7, 0), (8, 0), (1, 2 ** 31))),
        "b200q_release_sequences": ([16, 8, 16, 16, 16, 1, 3, 2, None], ((0, None), (2, None), (3, None), (4, None), (1, 0), (5, 0), (6, 0), (7, 0))),
        "b200q_copy_pages": ([one, 2, 64, None, 0, 0, 16, 16, 1, 8, 4, 16, 1 << 20, None], ((0, None), (0, null), (2, 0), (4, 1), (6, None), (7, None),
                             (8, 0), (9, 0), (10, 0))),
        "b200q_fork_sequences": ([one, 2, 64, one, 2, 8, 16, 8, 16, 16, 16, 16, 1, 3, 2, 4, 16, 1 << 20, None], ((0, null), (3, null), (5, 0), (6, None),
                                 (8, None), (9, None), (10, None), (11, None), (7, 0), (12, 0), (13, 0), (14, 0), (15, 0))),
        "b200q_compact_pages": ([one, 2, 64, one, 2, 8, 16, 8, 16, 3, 2, 4, 16, 16, 1 << 20, None], ((6, None), (8, None), (12, None), (7, 0), (9, 0),
                                (10, 0), (11, 0))),
    }
    for name, (good, changes) in cases.items():
        for i, v in changes:
            args = list(good)
            args[i] = v
            assert getattr(lib, name)(*args) == -1, (name, i, v)
    for name in ("b200q_reserve_pages", "b200q_copy_pages", "b200q_fork_sequences", "b200q_compact_pages"):
        for at, v in ((-3, None), (-2, 8)):              # no workspace, or one that is too small
            args = list(cases[name][0])
            args[at] = v
            assert getattr(lib, name)(*args) == -4, name
    args = list(cases["b200q_reserve_pages"][0])
    args[7] = (1 << 24) + 1
    assert lib.b200q_reserve_pages(*args) == -2


def test_fractions_of_tokens():
    pool, table, lengths = setup()
    with pytest.raises(TypeError):
        pages.reserve_pages(pool, table, lengths, 1.5)


def test_c_abi_refuses_workspaces_that_are_not_aligned():
    lib = cabi.load()
    one = (ctypes.c_void_p * 2)(16, 16)
    assert lib.b200q_reserve_pages(16, 8, 16, 16, None, 1, 3, 2, 4, 20, 1 << 20, None) == -4
    assert lib.b200q_copy_pages(one, 2, 64, None, 0, 0, 16, 16, 1, 8, 4, 20, 1 << 20, None) == -4
    assert lib.b200q_fork_sequences(one, 2, 64, one, 2, 8, 16, 8, 16, 16, 16, 16, 1, 3, 2, 4, 20, 1 << 20, None) == -4
    assert lib.b200q_compact_pages(one, 2, 64, one, 2, 8, 16, 8, 16, 3, 2, 4, 16, 20, 1 << 20, None) == -4
