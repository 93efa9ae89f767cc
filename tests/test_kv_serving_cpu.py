"""Host side of the cache's serving operators (tree decode, accumulated attention weight,
eviction by weight, keeping chosen positions): ancestor masks and refusals.  No GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

from ferrisres_b200 import _lib, kv
from ferrisres_b200._lib import ShapeError, UnsupportedError

CPU = torch.device("cpu")


def ancestors(parents):
    out = []
    for i, p in enumerate(parents):
        out.append((1 << i) | (out[p] if p >= 0 else 0))
    return out


@pytest.mark.parametrize("n", [1, 2, 5, 33, 64])
def test_tree_mask_is_the_ancestor_set(n):
    rng = np.random.default_rng(n)
    trees = [[-1] * n, list(range(-1, n - 1)), [int(rng.integers(-1, i)) if i else -1 for i in range(n)]]
    got = kv.tree_mask(trees, device="cpu")
    assert got.shape == (3, n) and got.dtype == torch.int64
    for t, row in zip(trees, got.tolist()):
        assert [m & (2**64 - 1) for m in row] == ancestors(t)
    assert kv.tree_mask(trees[2], device="cpu").tolist() == got[2].tolist()


@pytest.mark.parametrize("parents", [[], [0], [-1, 1], [-2], [-1] * 65, 3])
def test_tree_mask_refuses(parents):
    with pytest.raises(ShapeError):
        kv.tree_mask(parents, device="cpu")


def test_tree_arguments():
    q = torch.zeros((2, 3, 4, 128))
    m = torch.zeros((2, 3), dtype=torch.int64)
    for dtype in (torch.float32, torch.bfloat16):
        a, b, out = kv._tree_args(q.to(dtype), m[0], 2, CPU, None)
        assert out.dtype == dtype and out.shape == q.shape and b.shape == (2, 3)
    assert kv._tree_args(q, None, 2, CPU, None)[1] is None
    # a strided q is laid out, a misaligned one copied
    a, _, _ = kv._tree_args(torch.zeros((2, 3, 8, 128))[:, :, ::2], None, 2, CPU, None)
    assert a.is_contiguous()
    a, _, _ = kv._tree_args(torch.zeros(2 * 3 * 4 * 128 + 1)[1:].view(2, 3, 4, 128), None, 2, CPU, None)
    assert a.data_ptr() % 16 == 0
    for bad in (q.half(), q[0], torch.zeros((2, 3, 4, 64)), torch.zeros((3, 3, 4, 128))):
        with pytest.raises(ShapeError):
            kv._tree_args(bad, None, 2, CPU, None)
    for T in (0, 65):
        with pytest.raises(UnsupportedError):
            kv._tree_args(torch.zeros((2, T, 4, 128)), None, 2, CPU, None)
    for bad in (m.int(), m[:, :2], m[:1]):
        with pytest.raises(ShapeError):
            kv._tree_args(q, bad, 2, CPU, None)
    for bad in (q.bfloat16(), q[:, :2], torch.zeros((2, 3, 8, 128))[:, :, ::2]):
        with pytest.raises(ShapeError):
            kv._tree_args(q, m, 2, CPU, bad)


def test_index_lists():
    for shape, strides in (((5,), (0, 0)), ((2, 5), (5, 0)), ((2, 3, 5), (15, 5))):
        idx, n, s = kv._index_list(torch.zeros(shape, dtype=torch.int32), 2, 3, CPU)
        assert n == 5 and s == strides
    # 64-bit values that do not fit stay out of range instead of wrapping
    idx, _, _ = kv._index_list(torch.tensor([2**32 + 1, -(2**40), 7]), 2, 3, CPU)
    assert idx.tolist() == [2**31 - 1, -1, 7]
    for bad in (torch.zeros(5), torch.zeros((3, 5), dtype=torch.int32),
                torch.zeros((2, 2, 5), dtype=torch.int32), torch.tensor(3, dtype=torch.int32)):
        with pytest.raises(ShapeError):
            kv._index_list(bad, 2, 3, CPU)


def test_weight_rows():
    w = torch.zeros((2, 3, 10))
    assert kv._row_stride(w, (2, 3), 10, "w", CPU) == 10
    assert kv._row_stride(w[:, :, :7], (2, 3), 7, "w", CPU) == 10
    assert kv._row_stride(torch.zeros((1, 1, 9)), (1, 1), 4, "w", CPU) == 9
    assert kv._row_stride(torch.zeros((4, 10))[::2].unsqueeze(1), (2, 1), 10, "w", CPU) == 20
    for bad, least in ((w, 11), (w.double(), 4), (w[:, :2], 4), (w.transpose(0, 1), 4),
                       (w[:, :, ::2], 4), (w[0], 4), (torch.zeros((2, 3, 1)).expand(2, 3, 10), 4),
                       (torch.zeros((1, 3, 10)).expand(2, 3, 10), 4)):
        with pytest.raises(ShapeError):
            kv._row_stride(bad, (2, 3), least, "w", CPU)


def test_entry_points_refuse_null():
    L = _lib.lib()
    n = None
    f = C.c_float(0)
    for rc in (L.ft_flash_decode_3bit_weights(n, n, n, 1, f, n, n, 1, n),
               L.ft_kv3_tree_decode(n, n, 1, n, 0, 1, n, f, n, n),
               L.ft_kv_select_heavy(n, 1, 1, n, 1, n, 1, 1, 0, n, n, 0, n),
               L.ft_kv3_keep(n, n, 0, 1, n, 0, 0, n),
               L.ft_kvp_flash_decode_weights(n, n, 1, n, 1, n, 1, n, 1, f, n, n, 1, n),
               L.ft_kvp_tree_decode(n, n, 1, n, 1, n, 1, 1, 1, n, 0, 1, n, f, n, n),
               L.ft_kvp_keep(n, n, 1, n, 1, n, n, n, 1, n, 0, 0, n)):
        assert rc == 1 and b"null" in L.ft_last_error_string()


def test_select_needs_a_gpu_tensor():
    for bad in (torch.zeros((1, 1, 8)), [[[0.0] * 8]], None):
        with pytest.raises(ShapeError):
            kv.select_heavy(bad, 4)


def test_tree_arguments_of_other_kinds():
    q = torch.zeros((2, 3, 4, 128))
    for mask in ([[1, 2, 4]] * 2, 7):
        with pytest.raises(ShapeError):
            kv._tree_args(q, mask, 2, CPU, None)
    with pytest.raises(ShapeError):
        kv._tree_args(q, None, 2, CPU, q.numpy())
