"""Values that the C calls of the linear head's losses would see shortened or shifted are refused in Python."""

from __future__ import annotations

import pytest


@pytest.fixture(scope="module")
def kernels():
    from strideweave_b200 import build

    build.build()
    from strideweave_b200 import kernels

    return kernels


@pytest.mark.parametrize("value", [2 ** 32 - 100, 2 ** 31, -(2 ** 31) - 1])
def test_an_ignore_index_beyond_32_bits(kernels, value):
    with pytest.raises(ValueError, match="ignore_index must fit 32 bits"):
        kernels.linear_cross_entropy("Float32", 16, (8, 1), 16, (8, 1), 4, 10, 8, 16, ignore_index=value, loss_ptr=17)


@pytest.mark.parametrize("value", [2 ** 32 + 4, -(2 ** 32) + 4])
def test_a_number_of_entries_beyond_32_bits(kernels, value):
    with pytest.raises(ValueError, match="top_k must fit 32 bits"):
        kernels.linear_distillation("Float32", 16, (8, 1), 16, (8, 1), 4, 10, 8, 16, 16, value, loss_ptr=17)


@pytest.mark.parametrize("name, strides", [("h", dict(h=(8, 1, 1), w=(8,))), ("w", dict(w=(8, 1, 1))),
                                           ("dh", dict(dh=(8,), dw=(8, 1, 1))), ("dw", dict(dw=(1,)))])
def test_strides_are_pairs(kernels, name, strides):
    with pytest.raises(ValueError, match=f"^{name}_strides must be"):
        kernels.linear_cross_entropy("Float32", 16, strides.get("h", (8, 1)), 16, strides.get("w", (8, 1)), 4, 10, 8,
                                     16, loss_ptr=17, dh_ptr=16, dh_strides=strides.get("dh"), dw_ptr=16,
                                     dw_strides=strides.get("dw"))
