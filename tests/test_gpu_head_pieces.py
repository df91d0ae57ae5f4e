"""A step whose rows come in pieces, the weight's gradient added from piece to piece,
where a row of it is no whole number of vectors; and the weight's rows at any element."""
import pytest
import torch

from tests.test_gpu_head import check, inputs, rows_at

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D", [1, 23, 30, 36])
def test_columns_of_any_number(D, dtype):
    check(*inputs(65400, 70, D, dtype, seed=D, ignored=0.2), z=1e-3, what="pieces")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_at_any_element(dtype):
    check(*inputs(65400, 300, 41, dtype, seed=50, shift=3, pad=4, ignored=0.2), what="pieces of views")
