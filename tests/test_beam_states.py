"""The state arrays that zllm_amd.beam derives from tensors (no GPU): every
row's bytes are covered once, whatever the dimensions' order and cuts."""
import numpy as np
import pytest
import torch

from zllm_amd.beam import _blocks


def covered(t, d):
    """Byte offsets of every row as the descriptors have them."""
    rows = [[] for _ in range(t.shape[d])]
    for b in _blocks(t, d):
        start = b.d_base - t.data_ptr()
        for r in range(t.shape[d]):
            for o in range(b.n_outer):
                for i in range(b.n_inner):
                    at = start + r * b.row_stride + o * b.outer_stride + i * b.inner_stride
                    rows[r] += range(at, at + b.bytes)
    return rows


CASES = [
    lambda: (torch.zeros(2, 2, 6, 3, 5, 4, dtype=torch.bfloat16)[:, :, :, :, :3], 2),
    lambda: (torch.zeros(6, 7, dtype=torch.int32), 0),
    lambda: (torch.zeros(6, dtype=torch.int64), 0),
    lambda: (torch.zeros(5, 6), 1),
    lambda: (torch.zeros(4, 6, 8, dtype=torch.float16)[1:, :, 2:7], 1),
    lambda: (torch.zeros(3, 4, 6, 5, 4, 6)[:2, :3, :, :4, :3, :5], 2),
    lambda: (torch.zeros(3, 6, 4).permute(2, 1, 0), 1),
    lambda: (torch.zeros(1, 6, 1, 4), 1),
]


@pytest.mark.parametrize("make", CASES)
def test_rows_are_covered_once(make):
    t, d = make()
    size = t.element_size()
    got = covered(t, d)
    for r in range(t.shape[d]):
        row = t.select(d, r)
        offs = np.zeros(row.shape, np.int64) + (row.storage_offset() - t.storage_offset())
        for k in range(row.dim()):
            offs = offs + np.arange(row.shape[k]).reshape([-1 if j == k else 1 for j in range(row.dim())]) * row.stride(k)
        want = sorted(int(o) * size + b for o in offs.reshape(-1) for b in range(size))
        assert sorted(got[r]) == want


def test_adjacent_dimensions_are_one_block():
    t = torch.zeros(2, 2, 6, 3, 5, 4, dtype=torch.bfloat16)
    (b,) = _blocks(t, 2)
    assert (b.bytes, b.n_inner, b.n_outer) == (3 * 5 * 4 * 2, 4, 1)
    (b,) = _blocks(t[:, :, :, :, :2], 2)
    assert (b.bytes, b.n_inner, b.n_outer, b.inner_stride, b.row_stride) == (16, 3, 4, 40, 120)


def test_expanded_rows_are_refused():
    for t, d in ((torch.zeros(1, 4).expand(6, 4), 0), (torch.zeros(6, 1).expand(6, 4), 0)):
        with pytest.raises(ValueError):
            _blocks(t, d)
