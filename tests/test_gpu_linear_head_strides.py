"""Gradients of the linear head in every placement that reaches each element once."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from tests.test_gpu_linear_head import DTYPES, call, check, clean_status, reference, states  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def interleaved(x, sr, sc):
    """x at strides (sr, sc), rows and columns interleaved, and the storage around it."""
    rows, cols = x.shape
    base = torch.full(((rows - 1) * sr + (cols - 1) * sc + 1,), 9.0, dtype=x.dtype, device="cuda")
    view = base.as_strided((rows, cols), (sr, sc))
    view.copy_(x)
    return base, view


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("path", ["one call", "kept lse"])
@pytest.mark.parametrize("strides", [(49, 40), (40, 301), (98, 81)])
def test_interleaved_rows_and_columns(strides, path, dtype):
    T, V, D = 30, 300, 48
    h, w, y = states(T, V, D, dtype)
    up = torch.rand(T, device="cuda") + 0.5
    want = reference(h, w, up, targets=y)
    (_, hv), (_, wv) = interleaved(h, *strides), interleaved(w, *strides)
    (hb, dh), (wb, dw) = interleaved(torch.zeros_like(h), *strides), interleaved(torch.zeros_like(w), *strides)
    lse = call(h, w, targets=y, dh=None, dw=None)["lse"] if path == "kept lse" else None
    check(call(hv, wv, targets=y, up=up, dh=dh, dw=dw, lse_in=lse), want, dtype)
    dh.fill_(9.0)
    dw.fill_(9.0)
    assert bool((hb == 9.0).all()) and bool((wb == 9.0).all())
