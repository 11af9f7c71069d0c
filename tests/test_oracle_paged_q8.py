"""Pins of oracle/paged.py's 8-bit pages, worked out by hand."""
import numpy as np
import pytest

from oracle import paged as ref


def empty(blocks=1, nkv=1, block=16, hd=64, scale=127):
    return np.zeros((blocks, nkv, block, hd), np.int8), np.full((blocks, nkv, block // 16), scale, np.uint8)


def rows(values, hd=64):
    """[tokens, 1, hd] with one value each, the rest 0."""
    y = np.zeros((len(values), 1, hd))
    y[:, 0, 0] = values
    return y


@pytest.mark.parametrize("a,e", [(0.0, -24), (127.0, 0), (127.49, 0), (127.5, 1), (1.0, -6), (0.99609374, -7),
                                 (0.99609375, -6), (65279.9, 9), (65280.0, None), (np.inf, None), (1e-30, -24)])
def test_the_smallest_exponent(a, e):
    assert ref.exponent_q8(a) == e


def test_a_group_grows_and_its_rows_are_halved():
    codes, scale = ref.store_q8(*empty(), rows([100.0, -3.0]), [0, 1])
    assert scale[0, 0, 0] == 127 and codes[0, 0, :3, 0].tolist() == [100, -3, 0]
    codes, scale = ref.store_q8(codes, scale, rows([200.0]), [2])
    assert scale[0, 0, 0] == 128 and codes[0, 0, :3, 0].tolist() == [50, -2, 100]  # -1.5 to even
    codes, scale = ref.store_q8(codes, scale, rows([1.0]), [3])
    assert scale[0, 0, 0] == 128 and codes[0, 0, :4, 0].tolist() == [50, -2, 100, 0]  # 0.5 to even
    assert ref.values_q8(codes, scale)[0, 0, :4, 0].tolist() == [100.0, -4.0, 200.0, 0.0]


def test_the_first_row_starts_the_group_anew():
    codes, scale = ref.store_q8(*empty(), rows([100.0, -3.0]), [0, 1])
    codes, scale = ref.store_q8(codes, scale, rows([2.0, 1.0]), [3, 0])  # in any order
    assert scale[0, 0, 0] == 127 - 5
    assert codes[0, 0, :4, 0].tolist() == [32, 0, 0, 64]


def test_groups_heads_and_blocks_are_apart():
    codes, scale = empty(2, 2, 32, scale=103)
    y = np.zeros((2, 2, 64))
    y[0, 1], y[1, 0] = 3.0, np.nan
    codes, scale = ref.store_q8(codes, scale, y, [32 + 17, 5])
    assert scale[1, 1, 1] == 127 - 5 and codes[1, 1, 17, 0] == 96
    assert scale[0, 0, 0] == 255 and np.isnan(ref.values_q8(codes, scale)[0, 0, :16]).all()
    assert np.isfinite(ref.values_q8(codes, scale)[0, 0, 16:]).all()
    assert scale.tolist()[1][0] == [103, 103] and scale[0, 1].tolist() == [103, 103]
    codes, scale = ref.store_q8(codes, scale, np.zeros((1, 2, 64)), [4])
    assert scale[0, 0, 0] == 255  # until it starts anew
    codes, scale = ref.store_q8(codes, scale, np.zeros((1, 2, 64)), [0])
    assert scale[0, 0, 0] == 103


def test_slots_outside_are_not_stored():
    codes, scale = empty()
    c, s = ref.store_q8(codes, scale, rows([9.0, 9.0]), [-1, 16])
    assert np.array_equal(c, codes) and np.array_equal(s, scale)


def test_values_are_fp16_numbers():
    codes = np.tile(np.arange(-127, 128).astype(np.int8)[:, None], (1, 64))[None, None]
    codes = np.concatenate([codes, codes[:, :, :1]], 2)  # 256 rows
    for byte in (103, 104, 110, 127, 135, 136, 0, 200):
        v = ref.values_q8(codes, np.full((1, 1, 16), byte, np.uint8))
        assert np.array_equal(v, v.astype(np.float16).astype(np.float64))
