"""Types and sizes of the expert operators that the other tests leave out: 8-bit
products over every size, activation, stride and spread of groups within bounds that
hold for the instruction, and sums of f32 rows that go past the caches.

e4m3 values are whole numbers of -8 to 8: of their products the 8-bit instruction loses
nothing (a group of 8 sums to at most 512, and it keeps 13 bits below the largest), so
the bound of f32 sums in test_experts_gpu.py holds for them. For values of any size it
does not: the instruction may lose 2^-10 of the sum of the magnitudes."""
import pytest

import mini_triton_nvgpu_v1_amd as tb
import test_experts_tiles_gpu as tiles
from test_experts_gpu import SIZES, _check_rows, _counts, _gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("groups, slots, n, k", SIZES)
@pytest.mark.parametrize("spread", ["random", "last", "even"])
def test_8_bit_rows(device, groups, slots, n, k, spread):
    counts = _counts(spread, groups, slots, _gen(slots))
    _check_rows(groups, counts, slots, n, k, "f8", "bf16", tb.B_NK, gather=spread != "even",
                seed=slots, whole=True)


@pytest.mark.parametrize("act", [tb.ACT_RELU, tb.ACT_GELU_TANH, tb.ACT_SILU, tb.ACT_SWIGLU])
@pytest.mark.parametrize("c_dtype", ["f16", "f32"])
@pytest.mark.parametrize("groups, slots, n, k", [(6, 20, 72, 144), (4, 500, 152, 272),
                                                 (3, 1100, 264, 512)])
def test_8_bit_rows_activations(device, act, c_dtype, groups, slots, n, k):
    counts = _counts("random", groups, slots, _gen(3))
    _check_rows(groups, counts, slots, n, k, "f8", c_dtype, tb.B_NK, act, gather=True, whole=True)


@pytest.mark.parametrize("slots", [9, 60, 333, 900])
def test_8_bit_rows_strided(device, slots):
    counts = _counts("random", 5, slots - 4, _gen(4))  # the last slots have no group
    _check_rows(5, counts, slots, 136, 208, "f8", "f16", tb.B_NK, gather=True, pad=16,
                whole=True)


@pytest.mark.parametrize("slots", [1, 16, 17, 90, 600])
def test_8_bit_one_group_without_offsets(device, slots):
    _check_rows(1, [slots], slots, 392, 528, "f8", "f16", tb.B_NK, offsets=False, whole=True)


@pytest.mark.parametrize("tokens, top_k, width", [(4200, 4, 2048), (2100, 9, 2056)])
def test_combine_f32_past_the_caches(device, tokens, top_k, width):
    tiles.test_combine_past_the_caches(device, tokens, top_k, width, "f32")
