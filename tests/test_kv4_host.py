"""The 4-bit paged KV cache without a GPU: its definition (oracle/kv4_oracle.py) against
itself, the plain forms of perf/operators.py's layout, and the refusals that need no device."""

import ctypes

import numpy as np
import pytest
import torch

from llmnputest_b200 import _native, ops
from oracle import kv4_oracle as kv4


def test_every_byte_of_a_cell_has_one_meaning():
    used = np.zeros(kv4.CELL, int)
    np.add.at(used, kv4.CODE_AT[..., 0::2].reshape(-1), 1)
    np.add.at(used, (kv4.META_AT[..., None] + np.arange(4)).reshape(-1), 1)
    assert (used == 1).all()
    # no byte holds two tokens: a token's bytes are its own
    for which in range(2):
        owners = [set(kv4.CODE_AT[which, t]) for t in range(16)]
        assert sum(map(len, owners)) == len(set().union(*owners)) == 512


def test_pack_and_unpack():
    rng = np.random.default_rng(0)
    code = rng.integers(0, 16, (3, 2, 2, 16, 64)).astype(np.uint8)
    meta = kv4.bf16(rng.standard_normal((3, 2, 2, 16, 2)))
    cells = kv4.pack(code, meta)
    assert cells.shape == (3, 2, kv4.CELL)
    c, m = kv4.unpack(cells)
    assert np.array_equal(c, code) and np.array_equal(m, meta)


@pytest.mark.parametrize("x", [np.zeros(64), np.full(64, -3.0), np.arange(64.0), np.arange(64) * 1e-20,
                               np.linspace(-1e30, 1e30, 64), np.r_[np.zeros(63), 7.0]])
def test_quantise_keeps_within_its_step(x):
    code, (d, m) = kv4.quantise(np.asarray(x, np.float64))
    # m is off by a half step of bf16 at most, and so is d over 15 steps; inside, half a d
    slack = 2.0 ** -8 * (abs(m) + 16 * d) + 0.5 * d
    assert np.abs(code * d + m - x).max() <= slack


def test_quantise_marks_values_that_are_not_finite():
    x = np.zeros((3, 64))
    x[1, 5], x[2, 63] = np.nan, -np.inf
    code, meta = kv4.quantise(x)
    value = code * meta[..., :1] + meta[..., 1:]
    assert np.isfinite(value[0]).all() and np.isnan(value[1:]).all()


def test_oracle_rows_share_and_copy():
    """Two rows of one parent: the full page shared, the last one copied once."""
    table = np.array([[4, 2, -1], [0, -1, -1]], np.int32)
    lens, refs = np.array([20, 16], np.int32), np.array([1, 0, 1, 0, 1], np.int32)
    t, n, r, copies, info = kv4.reorder(table, lens, refs, np.array([0, 0]), 16, np.array([0, 20]))
    assert t.tolist() == [[4, 2, -1], [4, 0, 1]] and n.tolist() == [20, 20]
    assert r.tolist() == [1, 1, 1, 0, 2] and copies == [(2, 0)] and info.tolist() == [1, 1, 0, 0]
    t, r, moves, info = kv4.compact(t, r)
    assert t.tolist() == [[3, 2, -1], [3, 0, 1]] and r.tolist() == [1, 1, 1, 2, 0] and moves == [(4, 3)]
    assert info.tolist() == [4, 1, 0, 0]


def test_page_bytes():
    assert ops.kv4_page_bytes(64, 64) == 4 * 1152 and ops.kv4_page_bytes(16, 256) == 4 * 1152
    for bad in ((8, 64), (24, 64), (16, 96)):
        with pytest.raises(ValueError):
            ops.kv4_page_bytes(*bad)


def test_calls_fail_cleanly_without_a_device():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present; covered by the gpu tests")
    lib, n = _native.lib(), ctypes.c_size_t()
    shape = (1, 8, 64, 64, 4, 4)
    assert lib.b2_kv4_append(None, None, 512, 512, 1, None, None, None, None, None, *shape, 1e4, 0, None) == -4
    assert lib.b2_kv4_gather(None, None, 512, 512, 1, None, None, None, None, *shape, 0, None) == -4
    assert lib.b2_kv4_decode_workspace_size(1, 40, 8, 64, 64, 0, 256, ctypes.byref(n)) == -4
    assert lib.b2_kv4_decode(None, 2560, None, None, None, None, 0, 1, 40, 8, 64, 64, 4, 4, 256, 1e4, 0.125, None,
                             2560, None, 0, 0, None) == -4
    assert lib.b2_kv4_select(None, 2560, None, None, None, None, 2, 1, 40, 8, 64, 64, 4, 4, 256, 1e4, 0, None) == -4
    assert lib.b2_kv4_copy_pages(None, 4608, None, 0, 1, 4, None, None, 1, None) == -4
    assert lib.b2_kv4_reorder(None, 4608, None, 0, 1, 4, None, None, None, None, None, 1, 4, 64, None, None, None,
                              None, None, 0, None) == -4
    assert lib.b2_kv4_compact(None, 4608, None, 0, 1, 4, None, None, 1, 4, None, None, None, None, 0, None) == -4


def test_workspace_sizes():
    lib, n = _native.lib(), ctypes.c_size_t()
    assert lib.b2_kv4_reorder_workspace_size(4, 10, 100, ctypes.byref(n)) == 0 and n.value > 0
    assert lib.b2_kv4_reorder_workspace_size(0, 10, 100, ctypes.byref(n)) == -1
    assert lib.b2_kv4_compact_workspace_size(100, ctypes.byref(n)) == 0 and n.value >= 1200
    assert lib.b2_kv4_compact_workspace_size(100, None) == -1


def test_host_tensors_are_refused():
    pool = torch.zeros(4, 8, 4608, dtype=torch.uint8)
    table, pos = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 2560)
    heads = dict(n_kv_heads=8, head_dim=64)
    for call in (lambda: ops.kv4_append(x, x, pool, table, pos, **heads),
                 lambda: ops.kv4_gather(pool, table, pos, 1, **heads),
                 lambda: ops.kv4_decode(x, pool, table, pos, n_q_heads=40, **heads),
                 lambda: ops.kv4_select(x, torch.zeros(4, 8, 2, 64, dtype=torch.bfloat16), table, pos, n_q_heads=40,
                                        page=64, n_sel=2, **heads),
                 lambda: ops.kv4_copy_pages(pool[None], pos, pos),
                 lambda: ops.kv4_reorder(pool[None], table, pos, pos, pos, head_dim=64),
                 lambda: ops.kv4_compact(pool[None], table, pos)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
