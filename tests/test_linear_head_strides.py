"""Which strides of a gradient reach every element once, on the host: a call that passes this check is refused for
the next fault, a loss at an odd address."""

from __future__ import annotations

import itertools

import pytest


@pytest.fixture(scope="module")
def kernels():
    from strideweave_b200 import build

    build.build()
    from strideweave_b200 import kernels

    return kernels


def test_every_small_placement(kernels):
    for rows, cols, sr, sc in itertools.product((1, 2, 3, 5), (1, 2, 4, 7), range(0, 9), range(0, 9)):
        places = {i * sr + j * sc for i in range(rows) for j in range(cols)}
        with pytest.raises(ValueError, match="reach every element once|vector is not aligned") as refusal:
            kernels.linear_cross_entropy("Float32", 16, (cols, 1), 16, (cols, 1), rows, 10, cols, 16, loss_ptr=17,
                                         dh_ptr=16, dh_strides=(sr, sc))
        refused = "reach every element once" in str(refusal.value)
        assert refused == (len(places) != rows * cols), (rows, cols, sr, sc)
