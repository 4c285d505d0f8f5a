"""Arguments the linear head's losses refuse, on the host, before any device work."""

from __future__ import annotations

from ctypes import byref, c_void_p

import pytest


@pytest.fixture(scope="module")
def kernels():
    from strideweave_b200 import build

    build.build()
    from strideweave_b200 import kernels

    return kernels


def xent(kernels, *, dtype="BFloat16", h=16, hs=(64, 1), w=16, ws=(64, 1), tokens=4, vocab=100, dim=64, targets=16,
         **kw):
    kw.setdefault("loss_ptr", 16)
    return kernels.linear_cross_entropy(dtype, h, hs, w, ws, tokens, vocab, dim, targets, **kw)


def distill(kernels, *, index=16, logits=16, top_k=4, temperature=1.0, tokens=4, **kw):
    kw.setdefault("loss_ptr", 16)
    return kernels.linear_distillation("Float32", 16, (64, 1), 16, (64, 1), tokens, 100, 64, index, logits, top_k,
                                       temperature=temperature, **kw)


@pytest.mark.parametrize("kw, error, match", [
    (dict(dtype="Int32"), NotImplementedError, "no linear head kernel"),
    (dict(reduction="sum"), ValueError, "unknown reduction"),
    (dict(tokens=-1), ValueError, "tokens must be >= 0"),
    (dict(vocab=0), ValueError, "dim and vocab positive"),
    (dict(dim=0), ValueError, "dim and vocab positive"),
    (dict(tokens=1 << 31), NotImplementedError, "extents above"),
    (dict(tokens=1 << 30, vocab=1 << 30), NotImplementedError, "too many tiles"),
    (dict(workspace_limit=-1), ValueError, "negative workspace limit"),
    (dict(logit_scale=0.0), ValueError, "positive and finite"),
    (dict(logit_scale=-1.0), ValueError, "positive and finite"),
    (dict(logit_scale=float("nan")), ValueError, "positive and finite"),
    (dict(logit_scale=float("inf")), ValueError, "positive and finite"),
    (dict(loss_ptr=0), ValueError, "neither a loss nor a gradient"),
    (dict(loss_ptr=0, dh_ptr=16), ValueError, "needs the kept lse"),
    (dict(h=0), ValueError, "null states"),
    (dict(w=0), ValueError, "null weights"),
    (dict(targets=0), ValueError, "null targets"),
    (dict(hs=(-64, 1)), ValueError, "bad strides"),
    (dict(ws=(64, 1 << 60)), ValueError, "bad strides"),
    (dict(dh_ptr=16, dh_strides=(0, 1)), ValueError, "dh must reach every element once"),
    (dict(dw_ptr=16, dw_strides=(32, 1)), ValueError, "dw must reach every element once"),
    (dict(dw_ptr=16, dw_strides=(1, 50)), ValueError, "dw must reach every element once"),
    (dict(h=17), ValueError, "not aligned"),
    (dict(dtype="Float32", w=18), ValueError, "not aligned"),
    (dict(targets=18), ValueError, "vector is not aligned"),
    (dict(lse_ptr=17), ValueError, "vector is not aligned"),
])
def test_cross_entropy_refuses(kernels, kw, error, match):
    with pytest.raises(error, match=match):
        xent(kernels, **kw)


@pytest.mark.parametrize("kw, error, match", [
    (dict(top_k=0), ValueError, "1 to 256 teacher entries"),
    (dict(top_k=257), ValueError, "1 to 256 teacher entries"),
    (dict(temperature=0.0), ValueError, "temperature must be positive"),
    (dict(temperature=float("inf")), ValueError, "temperature must be positive"),
    (dict(temperature=1e-45), ValueError, "positive and finite"),
    (dict(index=0), ValueError, "null teacher entries"),
    (dict(logits=0), ValueError, "null teacher entries"),
    (dict(loss_ptr=0), ValueError, "neither a loss nor a gradient"),
])
def test_distillation_refuses(kernels, kw, error, match):
    with pytest.raises(error, match=match):
        distill(kernels, **kw)


def test_unknown_codes_and_a_null_plan(kernels):
    from strideweave_b200 import _native as N

    with pytest.raises(ValueError, match="null plan"):
        N.check(N.lib.sw_linear_xent(None, c_void_p(16), c_void_p(16), c_void_p(16), -100, 1.0, c_void_p(16), None,
                                     None, None, None, None))
    plan = N.LinearHead(7, 0, 4, 64, 100, 64, 1, 64, 1, 64, 1, 64, 1, 0)
    with pytest.raises(ValueError, match="unknown dtype"):
        N.check(N.lib.sw_linear_xent(byref(plan), c_void_p(16), c_void_p(16), c_void_p(16), -100, 1.0, c_void_p(16),
                                     None, None, None, None, None))
    plan = N.LinearHead(1, 7, 4, 64, 100, 64, 1, 64, 1, 64, 1, 64, 1, 0)
    with pytest.raises(ValueError, match="unknown reduction"):
        N.check(N.lib.sw_linear_xent(byref(plan), c_void_p(16), c_void_p(16), c_void_p(16), -100, 1.0, c_void_p(16),
                                     None, None, None, None, None))
