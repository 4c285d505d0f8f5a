"""The linear head's losses at sizes that take the paths of larger calls, against binary64 (tolerances as in
test_gpu_linear_head.py): a last wave of gradient tiles cut along K after whole ones, logits computed again by CTA
pairs, remainder rows of the logits computed again, many more rows than count, more rows than one scan of the flags
takes at 8 a CTA, and results that TMA cannot write."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from tests.test_gpu_linear_head import DTYPES, call, check, clean_status, reference, states, teacher  # noqa: E402, F401
from tests.test_gpu_linear_head_rows import row_errors  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F32 = DTYPES


def counted(T, count, seed=5):
    """Which rows count: `count` of them, anywhere."""
    g = torch.Generator().manual_seed(seed)
    keep = torch.zeros(T, dtype=torch.bool)
    keep[torch.randperm(T, generator=g)[:count]] = True
    return keep.cuda()


def loss_arguments(op, T, V, y, keep):
    if op == "xent":
        return dict(targets=torch.where(keep, y, torch.full_like(y, -100)))
    index, logits = teacher(T, V, 7, empty=False)
    index[~keep] = -1
    return dict(index=index, logits=logits, tau=2.0)


def run(dtype, T, V, D, count, path, op="xent", mean=False, rows=True):
    h, w, y = states(T, V, D, dtype)
    kw = loss_arguments(op, T, V, y, counted(T, count))
    up = torch.rand(1 if mean else T, device="cuda") + 0.5
    want = reference(h, w, up, mean=mean, **kw)
    first = call(h, w, mean=mean, up=up, limit=1 if path == "pieces" else 0, **kw)
    check(first, want, dtype, mean)
    out = first
    if path == "kept lse":
        out = call(h, w, mean=mean, up=up, lse_in=first["lse"], **kw)
        check(out, want, dtype, mean)
    if rows:  # no row of a gradient is far off on its own: a tile or a part in the wrong place would be
        for name, expect in (("dh", want[2]), ("dw", want[3])):
            assert float(row_errors(out[name], expect).max()) <= 0.05, name


@pytest.mark.parametrize("path", ["one call", "kept lse"])
@pytest.mark.parametrize("dtype,T,V,D,count", [
    (BF16, 5000, 9000, 1030, 5000), (F32, 5000, 9000, 1030, 5000),     # dh: 74 tiles, then 26 in 2 parts
    (BF16, 5000, 9000, 1030, 4800), (F32, 5000, 9000, 1030, 2600), (BF16, 5000, 9000, 1030, 60),
    (BF16, 9500, 10000, 1030, 9500),                                   # dh in tall tiles, the rest in 3 parts
    (F32, 3000, 4000, 1500, 3000), (F32, 3000, 4000, 1500, 700),       # dw: 74 tiles, then 22 in 3 parts
    (BF16, 3600, 3750, 1030, 3600), (BF16, 3600, 3750, 1030, 900),     # dw in 4 parts
])
def test_a_last_wave_cut_along_k(dtype, T, V, D, count, path):
    run(dtype, T, V, D, count, path)


@pytest.mark.parametrize("op", ["xent", "distill"])
@pytest.mark.parametrize("path", ["kept lse", "pieces"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V,D,count", [(700, 6000, 520, 700), (700, 6000, 520, 333), (1, 500, 72, 1),
                                         (40, 900, 72, 40), (64, 900, 130, 64), (65, 900, 130, 65),
                                         (500, 900, 72, 40), (500, 900, 72, 64), (500, 900, 72, 1),
                                         (2000, 3000, 264, 64), (64, 700, 2100, 64)])
def test_logits_computed_again(T, V, D, count, dtype, path, op):
    run(dtype, T, V, D, count, path, op)


@pytest.mark.parametrize("op", ["xent", "distill"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mean", [False, True])
@pytest.mark.parametrize("T,count", [(16385, 16385), (17001, 5000), (20000, 50)])
def test_more_than_16384_rows(T, count, mean, dtype, op):
    run(dtype, T, 700, 72, count, "one call", op, mean)


@pytest.mark.parametrize("path", ["one call", "kept lse"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_column_major_states_of_more_than_16384_rows(dtype, path):
    T, V, D = 16500, 300, 65
    h, w, y = states(T, V, D, dtype)
    kw = dict(targets=torch.where(counted(T, 9000), y, torch.full_like(y, -100)))
    up = torch.rand(T, device="cuda") + 0.5
    want = reference(h, w, up, **kw)
    h = h.t().contiguous().t()
    dh = torch.full((D, T), 7.0, dtype=dtype, device="cuda").t()
    lse = call(h, w, dh=None, dw=None, **kw)["lse"] if path == "kept lse" else None
    check(call(h, w, up=up, dh=dh, lse_in=lse, **kw), want, dtype)
