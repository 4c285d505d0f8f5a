"""What a call of the linear head's losses takes from the device's pool stays within its workspace limit, and the
results of the plans that smaller limits lead to are the same."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from tests.test_gpu_linear_head import DTYPES, call, check, clean_status, reference, states, teacher  # noqa: E402, F401

pytestmark = pytest.mark.gpu

MB = 1 << 20


def peak(run):
    """Bytes that `run` held in the device's default memory pool at most, and its result."""
    from cuda.bindings import driver as drv

    from strideweave_b200 import _native as N

    torch.cuda.synchronize()
    _, dev = drv.cuDeviceGet(N.current_device())
    _, pool = drv.cuDeviceGetDefaultMemPool(dev)
    kind = drv.CUmemPool_attribute
    (err,) = drv.cuMemPoolSetAttribute(pool, kind.CU_MEMPOOL_ATTR_USED_MEM_HIGH, drv.cuuint64_t(0))
    assert err == drv.CUresult.CUDA_SUCCESS
    before = int(drv.cuMemPoolGetAttribute(pool, kind.CU_MEMPOOL_ATTR_USED_MEM_CURRENT)[1])
    out = run()
    torch.cuda.synchronize()
    err, high = drv.cuMemPoolGetAttribute(pool, kind.CU_MEMPOOL_ATTR_USED_MEM_HIGH)
    assert err == drv.CUresult.CUDA_SUCCESS
    return int(high) - before, out


@pytest.mark.parametrize("mode", ["train", "kept lse"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_scratch_stays_within_its_limit(dtype, mode):
    T, V, D = 3000, 5000, 256
    h, w, y = states(T, V, D, dtype)
    y[7] = -100
    up = torch.rand(T, device="cuda") + 0.5
    lse = call(h, w, targets=y, dh=None, dw=None)["lse"] if mode == "kept lse" else None
    want = reference(h, w, up, targets=y)
    free, _ = peak(lambda: call(h, w, targets=y, up=up, lse_in=lse))
    seen = set()
    for limit in (256 * MB, 96 * MB, 64 * MB, 48 * MB, 32 * MB, 24 * MB, 20 * MB):
        took, out = peak(lambda: call(h, w, targets=y, up=up, lse_in=lse, limit=limit))
        check(out, want, dtype)
        assert took <= max(limit, 20 * MB)
        seen.add(took)
    assert max(seen) == free  # nothing was asked of the largest limit
    assert len(seen) >= 4


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("op", ["xent", "distill"])
@pytest.mark.parametrize("mean", [False, True])
def test_blocks_of_rows_with_their_sums(dtype, op, mean):
    """A limit under which the exponentials go in three blocks, the last ones reached by no row or by few."""
    T, V, D = 3300, 2000, 72
    h, w, y = states(T, V, D, dtype)
    up = torch.rand(1 if mean else T, device="cuda") + 0.5
    limit = 10 * MB if dtype == torch.bfloat16 else 17 * MB
    for ignored in (slice(0, 0), slice(1200, 3300), slice(40, 3300)):
        kw = dict(targets=y.clone())
        kw["targets"][ignored] = -100
        if op == "distill":
            index, logits = teacher(T, V, 20)
            index[ignored] = -1
            kw = dict(index=index, logits=logits, tau=2.0)
        took, out = peak(lambda: call(h, w, up=up, mean=mean, limit=limit, **kw))
        assert took <= limit
        check(out, reference(h, w, up, mean=mean, **kw), dtype, mean)


@pytest.mark.parametrize("dtype", DTYPES)
def test_statistics_in_blocks_of_rows(dtype):
    """A loss alone, its statistics 1024 rows and more at a time."""
    T, V, D = 5000, 9000, 64
    h, w, y = states(T, V, D, dtype)
    y[::3] = -100
    up = torch.ones(T, device="cuda")
    want = reference(h, w, up, targets=y)
    free, _ = peak(lambda: call(h, w, targets=y, dh=None, dw=None))
    limit = 4 * MB if dtype == torch.bfloat16 else 8 * MB
    assert free > limit
    took, out = peak(lambda: call(h, w, targets=y, dh=None, dw=None, limit=limit))
    assert took <= limit
    check(out, want, dtype)
