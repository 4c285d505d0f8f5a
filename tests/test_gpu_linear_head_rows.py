"""Each row's gradient of the linear head's losses against binary64, where one tolerance for a whole
matrix would hide a row: rows sure of their target, and rows far larger than the others.

Tolerances, from the arithmetic and before any run, relative to the row's own norm:

- A logit is off by at most 1e-5 of the largest, so a small probability by 1e-5 (1 + max |s|) of itself.
- In a row whose target has probability 1 - q the target's entry of the logits' gradient is -q.  The sum
  of the row's exponentials is 1 + q and off by a few 2^-24, so that q is by 2^-22 / q of itself.
- Gradients from a kept lse: its rounding, 2^-24 |lse|, is an absolute error of a logit.
- bf16: the logits' gradient and the result are each rounded to 8 bits: 2^-8 together.
"""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

from tests.test_gpu_linear_head import DTYPES, call, clean_status, reference, states  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def row_errors(got, want):
    """Of every row, the error's norm relative to the row's (rows of zeros: absolute)."""
    n, d = want.norm(dim=1), (got.double() - want).norm(dim=1)
    return torch.where(n > 0, d / n.clamp(min=1e-300), d)


def sure_rows(T, V, D, dtype, gap):
    """Rows whose logits are about 60 at the target, 60 - gap at one other word and near 0 elsewhere."""
    g = torch.Generator().manual_seed(3)
    w = (torch.randn(V, D, generator=g) / math.sqrt(D)).to(dtype).cuda()
    y = torch.arange(T, device="cuda")
    a, b = w[y].float(), w[y + T].float()
    h = 60 * a / a.square().sum(1, keepdim=True) + (60 - gap) * b / b.square().sum(1, keepdim=True)
    return h.to(dtype), w, y.to(torch.int32)


@pytest.mark.parametrize("path", ["one call", "kept lse", "pieces"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap", [5.0, 7.0, 9.0])
@pytest.mark.parametrize("T", [40, 200])
def test_gradients_of_rows_sure_of_their_target(dtype, T, gap, path):
    V, D = 600, 2048
    h, w, y = sure_rows(T, V, D, dtype, gap)
    up = torch.rand(T, device="cuda") + 0.5
    loss, lse, dh, dw, _, top = reference(h, w, up, targets=y)
    if path == "kept lse":
        kept = call(h, w, targets=y, dh=None, dw=None)["lse"]
        out = call(h, w, targets=y, up=up, lse_in=kept)
    else:
        out = call(h, w, targets=y, up=up, limit=1 if path == "pieces" else 0)
    q = 1 - torch.exp(-loss)
    assert 1e-6 < float(q.min()) and float(q.max()) < 0.5
    tol = 1e-5 * (1 + top) + 2.0 ** -22 / q
    if path == "kept lse":
        tol = tol + 2.0 ** -24 * lse / q
    if dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8
    assert bool((row_errors(out["dh"], dh) <= tol).all())
    rows = y.long()
    assert bool((row_errors(out["dw"][rows], dw[rows]) <= tol).all())
    assert bool((row_errors(out["dw"][rows + T], dw[rows + T]) <= tol).all())


@pytest.mark.parametrize("path", ["one call", "kept lse", "pieces"])
def test_a_row_of_huge_logits_is_finite_and_stays_alone(path):
    """One row's logits are about 1e14: its softmax is one word, its loss a difference of two logits."""
    T, V, D = 70, 500, 64
    dtype = torch.bfloat16
    h, w, y = states(T, V, D, dtype)
    h[3] = (h[3].float() * 1e13).to(dtype)
    up = torch.ones(T, device="cuda")
    loss, lse, dh, dw, _, _ = reference(h, w, up, targets=y)
    first = call(h, w, targets=y, up=up, limit=1 if path == "pieces" else 0)
    top = (h.double() @ w.double().t()).abs().amax(1)
    assert bool(((first["loss"].double() - loss).abs() <= 1e-5 * (1 + top)).all())
    assert bool(((first["lse"].double() - lse).abs() <= 1e-5 * (1 + top)).all())
    out = call(h, w, targets=y, up=up, lse_in=first["lse"]) if path == "kept lse" else first
    others = top[torch.arange(T, device="cuda") != 3].max()
    tol = 2.0 ** -8 + 1e-5 * (1 + float(others))
    assert bool((row_errors(out["dh"], dh) <= tol).all())
    assert bool((row_errors(out["dw"], dw) <= tol).all())


def columns(x):
    return x.t().contiguous().t()


@pytest.mark.parametrize("path", ["one call", "kept lse", "pieces"])
@pytest.mark.parametrize("kind", ["a state of 1e13", "states of 1e9", "a word of 1e9", "factors from 1e-6",
                                  "factors from 1e-12", "all"])
@pytest.mark.parametrize("T,V,D,layout", [(60, 700, 96, "rows"), (300, 3000, 200, "rows"), (60, 700, 96, "columns"),
                                          (40, 9600, 65, "columns")])
def test_float32_rows_far_apart(T, V, D, layout, kind, path):
    """What one row holds is no other row's loss: states, words and upstream factors 1e6 to 1e13 apart."""
    h, w, y = states(T, V, D, torch.float32)
    h[:, 0] = 1.0 + h[:, 0].abs()
    up = torch.rand(T, device="cuda") + 0.5
    big = torch.zeros(T, dtype=torch.bool, device="cuda")
    if kind in ("a state of 1e13", "all"):
        big[7] = True
        h[7] *= 1e13
    if kind == "states of 1e9":
        big[2::3] = True
        h[big] *= 1e9
    if kind in ("a word of 1e9", "all"):  # never likely: its logits are below -1e9
        y[y == 11] = 12
        w[11] = 0.0
        w[11, 0] = -1e9
    if kind.startswith("factors") or kind == "all":
        up = torch.logspace(-6 if kind.endswith("1e-6") else -12, 0, T, device="cuda")
    if layout == "columns":
        h, w = columns(h), columns(w)
    loss, lse, dh, dw, _, _ = reference(h, w, up, targets=y)
    out = call(h, w, targets=y, up=up, limit=1 if path == "pieces" else 0)
    s = (h.double() @ w.double().t()).abs()
    touched = s.argmax(1)[big]  # words whose gradient the large states are
    s[:, 11] = 0.0
    top = s.amax(1)
    assert bool(((out["loss"].double() - loss).abs() <= 1e-5 * (1 + top)).all())
    assert bool(((out["lse"].double() - lse).abs() <= 1e-5 * (1 + top)).all())
    if path == "kept lse":
        out = call(h, w, targets=y, up=up, lse_in=out["lse"])
    assert bool(torch.isfinite(out["dh"]).all()) and bool(torch.isfinite(out["dw"]).all())
    tol = 2e-5 * (1 + top / 4)
    assert bool((row_errors(out["dh"], dh) <= tol)[~big].all())
    words = torch.ones(V, dtype=torch.bool, device="cuda")
    words[touched] = False
    words[y[big].long()] = False
    assert bool((row_errors(out["dw"], dw) <= float(tol[~big].max()))[words].all())
