"""Logits of a 4-bit head against the formula in 64 bits at every number of ids at
which the kernels take another number of tiles a wave, or of waves along the columns.
The tolerance is tests/test_gpu_q4.py's."""
import pytest
import torch

from tests.test_gpu_q4 import bound, check, parts, states, weight  # noqa: F401

pytestmark = pytest.mark.gpu


# 33 to 64 rows of a 16-bit type: 1, 2, 3, 4, 5 (groups of 32 without minima) and 4 tiles a wave
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("V", [16384, 16385, 65536, 65537, 98304, 98305, 131072, 131073, 163840, 163841])
def test_tiles_a_wave(V, group, mins, dtype):
    check(64 if V % 2 else 37, V, 3 * group, group, mins, dtype)


# rows of any type that two tiles of 32 rows take, over the same ids
@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("B,dtype", [(17, "f32"), (33, "f32"), (64, "f32"), (32, "f16"), (20, "bf16")])
def test_tiles_of_32_rows(B, dtype, mins):
    for V in (16385, 65537, 140001):
        check(B, V, 192, 64, mins, dtype)


# one wave along the columns, up to 16 rows
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("B", [1, 4, 5, 8, 9, 16])
def test_one_wave_along_the_columns(B, group, mins, dtype):
    for V in (65520, 65521, 70001):
        check(B, V, 3 * group, group, mins, dtype)


def test_steps_of_columns():
    """1 to 8 steps of 128 columns: the three stages' last turn, for each width."""
    for n in range(1, 9):
        for V in (1000, 20000, 90000, 120000, 150000):
            check(50, V, 128 * n, 32, False, "bf16")
        check(100, 2000, 128 * n, 128, True, "f16")
