"""Cross entropy and distillation of a linear head against their formulas in binary64.

Tolerances, from the arithmetic and before any run:

- loss and lse.  Products are exact (bf16) or carry 22 bits (Float32), and a
  tensor-core sum of 512 products loses at most 2^-23 of its running value in
  each of 96 steps, so a logit is off by at most 1e-5 of the largest logit (and
  at least one rounding of Float32): 1e-5 (1 + max |s|), absolute.
- Float32 gradients: a softmax off by the logits' error, 1e-5 (1 + max |s|) of
  itself, and products of 22 bits: 2e-5 (1 + max |s| / 4) in the Frobenius norm.
- bf16 gradients: the logits' gradient and the result are each rounded once to
  8 bits, an rms error of 2^-8 / sqrt(3) at most, together 3.2e-3, and the
  terms of a sum do not cancel systematically: 5e-3 in the Frobenius norm.
  Where a case makes them cancel it says so and scales by the terms' norm.
"""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

IGNORE = -100


@pytest.fixture(autouse=True)
def clean_status():
    from strideweave_b200 import _native as N

    N.device_status()
    yield
    assert N.device_status() == N.SW_OK


def states(T, V, D, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, D, generator=g) / math.sqrt(D)).to(dtype).cuda()
    y = torch.randint(0, V, (T,), generator=g).cuda()
    h = torch.randn(T, D, generator=g).cuda() * scale + 6 * torch.rand(T, 1, generator=g).cuda() * w[y].float()
    return h.to(dtype), w, y.to(torch.int32)


def teacher(T, V, K, seed=0, empty=True):
    g = torch.Generator().manual_seed(seed + 1)
    index = torch.stack([torch.randperm(V, generator=g)[:K] if K <= V else torch.randint(0, V, (K,), generator=g)
                         for _ in range(T)]) if T else torch.zeros(0, K, dtype=torch.long)
    logits = 3 * torch.randn(T, K, generator=g)
    if empty and T > 2:
        index[1] = -1
        logits[2, K // 2:] = -math.inf
    return index.to(torch.int32).cuda(), logits.cuda()


def reference(h, w, up, *, targets=None, index=None, logits=None, tau=1.0, scale=None, mean=False, lse_in=None):
    """loss (per row), lse, dh, dw in binary64; the rows that count; max |s|."""
    T, V = h.shape[0], w.shape[0]
    scale = 1.0 / tau if scale is None else scale
    h, w = h.double(), w.double()
    if targets is not None:
        index, p = targets.long()[:, None], (targets != IGNORE).double()[:, None]
        there = targets[:, None] != IGNORE
    else:
        there = (index >= 0) & (logits != -math.inf)
        t = torch.where(there, logits.double() / tau, torch.tensor(-math.inf, dtype=torch.float64, device="cuda"))
        p = torch.nan_to_num(torch.softmax(t, 1), nan=0.0)
        index = index.long()
    rows = there.any(1)
    hz = torch.where(rows[:, None], h, torch.zeros_like(h))
    s = scale * hz @ w.t()
    lse = torch.logsumexp(s, 1) if lse_in is None else lse_in.double()
    target = torch.zeros(T, V, dtype=torch.float64, device="cuda").scatter_add_(1, index.clamp(min=0), p)
    ent = torch.xlogy(p, p).sum(1)
    loss = torch.where(rows, tau ** 2 * (ent + lse - (target * s).sum(1)), torch.zeros_like(lse))
    up = (up.double() / rows.sum()).expand(T) if mean else up.double()
    g = (torch.exp(s - lse[:, None]) - target) * (up * scale * tau ** 2)[:, None]
    g = torch.where(rows[:, None], g, torch.zeros_like(g))
    top = float(s[rows].abs().max()) if bool(rows.any()) else 0.0
    return loss, torch.where(rows, lse, torch.zeros_like(lse)), g @ w, g.t() @ hz, rows, top


def call(h, w, *, targets=None, index=None, logits=None, tau=1.0, scale=1.0, mean=False, up=None, dh="new", dw="new",
         lse_in=None, limit=0, stream=0):
    from strideweave_b200 import kernels

    T, D = h.shape
    V = w.shape[0]
    out = {}
    kw = dict(reduction="mean" if mean else "none", workspace_limit=limit, stream=stream,
              upstream_ptr=up.data_ptr() if up is not None else 0)
    if lse_in is None:
        out["loss"] = torch.full((1,) if mean else (T,), 7.0, device="cuda")
        out["lse"] = torch.full((T,), 7.0, device="cuda")
        kw.update(loss_ptr=out["loss"].data_ptr(), lse_ptr=out["lse"].data_ptr())
    else:
        kw.update(lse_ptr=lse_in.data_ptr())
    for name, like, given in (("dh", h, dh), ("dw", w, dw)):
        if given is None:
            continue
        g = torch.full(like.shape, 7.0, dtype=like.dtype, device="cuda") if isinstance(given, str) else given
        out[name] = g
        kw.update({name + "_ptr": g.data_ptr(), name + "_strides": g.stride()})
    head = ("BFloat16" if h.dtype == torch.bfloat16 else "Float32", h.data_ptr(), h.stride(), w.data_ptr(), w.stride(),
            T, V, D)
    if targets is not None:
        kernels.linear_cross_entropy(*head, targets.data_ptr(), ignore_index=IGNORE, logit_scale=scale, **kw)
    else:
        kernels.linear_distillation(*head, index.data_ptr(), logits.data_ptr(), index.shape[1], temperature=tau, **kw)
    return out


def frobenius(got, want):
    n = float(want.norm())
    return float((got.double() - want).norm()) / n if n else float(got.double().abs().max())


def check(out, want, dtype, mean=False):
    loss, lse, dh, dw, rows, top = want
    tol = 1e-5 * (1 + top)
    if "loss" in out:
        expect = loss.sum() / rows.sum() if mean else loss
        assert float((out["loss"].double() - expect).abs().max()) <= 4 * tol  # tau^2 is 4 at most here
        assert float((out["lse"].double() - lse).abs().max()) <= tol
    gtol = 5e-3 if dtype == torch.bfloat16 else 2e-5 * (1 + top / 4)
    for name, expect in (("dh", dh), ("dw", dw)):
        if name in out:
            assert bool(torch.isfinite(out[name]).all())
            assert frobenius(out[name], expect) <= gtol, name


DTYPES = [torch.bfloat16, torch.float32]
SIZES = [(1, 2, 8), (2, 31, 3), (3, 300, 64), (33, 257, 65), (127, 255, 128), (128, 256, 64), (129, 513, 72),
         (300, 1000, 136), (260, 700, 1030), (64, 4099, 520), (1, 5000, 1024)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V,D", SIZES)
@pytest.mark.parametrize("mean", [False, True])
def test_cross_entropy(T, V, D, dtype, mean):
    h, w, y = states(T, V, D, dtype)
    y[torch.arange(T, device="cuda") % 5 == 3] = IGNORE
    up = torch.rand(1 if mean else T, device="cuda") + 0.5
    out = call(h, w, targets=y, mean=mean, up=up)
    check(out, reference(h, w, up, targets=y, mean=mean), dtype, mean)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V,D,K", [(1, 40, 8, 3), (5, 300, 64, 1), (33, 257, 65, 7), (130, 513, 72, 32),
                                     (300, 1000, 136, 64), (40, 700, 264, 256), (7, 4099, 520, 129), (3, 2, 16, 2)])
@pytest.mark.parametrize("mean", [False, True])
def test_distillation(T, V, D, K, dtype, mean):
    h, w, _ = states(T, V, D, dtype)
    index, logits = teacher(T, V, K)
    up = torch.rand(1 if mean else T, device="cuda") + 0.5
    out = call(h, w, index=index, logits=logits, tau=2.0, mean=mean, up=up)
    check(out, reference(h, w, up, index=index, logits=logits, tau=2.0, mean=mean), dtype, mean)


@pytest.mark.parametrize("dtype", DTYPES)
def test_entries_at_tile_borders_and_repeated_columns(dtype):
    T, V, D = 6, 1030, 64
    h, w, _ = states(T, V, D, dtype)
    cols = [0, 31, 32, 63, 127, 128, 255, 256, 257, 511, 512, 767, 768, 1023, 1024, 1029, 1029, 0, 512, 5000000]
    index = torch.tensor([cols[i:] + cols[:i] for i in range(T)], dtype=torch.int32, device="cuda")
    index[index == 5000000] = -3  # a negative column is no entry, whatever its logit
    logits = torch.linspace(2, -2, len(cols), device="cuda").expand(T, -1).contiguous()
    up = torch.ones(T, device="cuda")
    out = call(h, w, index=index, logits=logits, tau=1.0, up=up)
    check(out, reference(h, w, up, index=index, logits=logits, tau=1.0), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_entropy_targets_at_tile_borders(dtype):
    V, D = 1030, 64
    cols = torch.tensor([0, 31, 32, 127, 128, 255, 256, 511, 512, 1023, 1024, 1029], dtype=torch.int32, device="cuda")
    h, w, _ = states(len(cols), V, D, dtype)
    up = torch.ones(len(cols), device="cuda")
    check(call(h, w, targets=cols, up=up), reference(h, w, up, targets=cols), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("op", ["xent", "distill"])
def test_rows_that_do_not_count_are_never_read(op, dtype):
    T, V, D = 150, 600, 72
    h, w, y = states(T, V, D, dtype)
    out_of = torch.arange(T, device="cuda") % 3 != 1
    kw = dict(targets=torch.where(out_of, torch.full_like(y, IGNORE), y))
    if op == "distill":
        index, logits = teacher(T, V, 4, empty=False)
        index[out_of] = -1
        logits[out_of] = math.nan  # what an absent entry holds does not matter
        kw = dict(index=index, logits=logits, tau=1.5)
    up = torch.ones(T, device="cuda")
    want = reference(h, w, up, **kw) if op == "xent" else reference(
        h, w, up, index=index, logits=torch.nan_to_num(logits, nan=0.0), tau=1.5)
    h = h.clone()
    h[out_of] = torch.tensor([math.nan, math.inf, -math.inf] * 24, dtype=dtype, device="cuda")[:D]
    up = torch.where(out_of, torch.full_like(up, math.nan), up)
    out = call(h, w, up=up, **kw)
    check(out, want, dtype)
    assert bool((out["loss"][out_of] == 0).all()) and bool((out["lse"][out_of] == 0).all())
    assert bool((out["dh"][out_of] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mean", [False, True])
def test_no_row_counts(dtype, mean):
    h, w, y = states(9, 300, 72, dtype)
    y[:] = IGNORE
    out = call(h, w, targets=y, mean=mean)
    assert bool(out["loss"].isnan().all()) if mean else bool((out["loss"] == 0).all())
    for name in ("lse", "dh", "dw"):
        assert bool((out[name] == 0).all()), name
    index, logits = teacher(9, 300, 4)
    out = call(h, w, index=torch.full_like(index, -1), logits=logits, tau=2.0, mean=mean)
    for name in ("lse", "dh", "dw"):
        assert bool((out[name] == 0).all()), name


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_rows_at_all(dtype):
    h, w, y = states(1, 300, 72, dtype)
    out = call(h[:0], w, targets=y[:0], mean=True)
    assert bool(out["loss"].isnan().all()) and bool((out["dw"] == 0).all())
    out = call(h[:0], w, targets=y[:0])
    assert bool((out["dw"] == 0).all())


def test_a_target_outside_the_vocabulary_is_reported():
    from strideweave_b200 import _native as N

    h, w, y = states(6, 300, 72, torch.bfloat16)
    for bad in (300, -1, 2**31 - 1):
        wrong = y.clone()
        wrong[2] = bad
        ignored = y.clone()
        ignored[2] = IGNORE
        up = torch.ones(6, device="cuda")
        out = call(h, w, targets=wrong, up=up)
        assert N.device_status() == N.SW_ERR_INVALID
        assert bool(out["loss"][2].isnan()) and int(out["loss"].isnan().sum()) == 1
        want = reference(h, w, up, targets=ignored)
        out["loss"][2] = 0.0
        check(out, want, torch.bfloat16)
        assert bool(call(h, w, targets=wrong, mean=True)["loss"].isnan().all())
        assert N.device_status() == N.SW_ERR_INVALID
    index, logits = teacher(6, 300, 4, empty=False)
    outside = index.clone()
    outside[3, 1] = 300
    out = call(h, w, index=outside, logits=logits, up=up)
    assert N.device_status() == N.SW_ERR_INVALID
    outside[3, 1] = -1
    check(out, reference(h, w, up, index=outside, logits=logits), torch.bfloat16)


def placed(x, kind):
    """x in another placement, and the storage around it."""
    rows, cols = x.shape
    if kind == "columns":
        base = torch.full((cols, rows + 3), 9.0, dtype=x.dtype, device="cuda")
        view = base.t()[:rows]
    elif kind == "pitch":
        base = torch.full((rows, cols + 5), 9.0, dtype=x.dtype, device="cuda")
        view = base[:, 2:2 + cols]
    elif kind == "aligned pitch":
        base = torch.full((rows, (cols + 23) // 8 * 8), 9.0, dtype=x.dtype, device="cuda")
        view = base[:, 8:8 + cols]
    elif kind == "offset":
        base = torch.full((rows * cols + 1,), 9.0, dtype=x.dtype, device="cuda")
        view = base[1:].view(rows, cols)
    else:  # both strides above one
        base = torch.full((rows, 2 * cols + 1), 9.0, dtype=x.dtype, device="cuda")
        view = base[:, :2 * cols:2]
    view.copy_(x)
    return base, view


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 75])
@pytest.mark.parametrize("kind", ["columns", "pitch", "aligned pitch", "offset", "strided"])
def test_placements(kind, D, dtype):
    T, V = 140, 390
    h, w, y = states(T, V, D, dtype)
    y[5] = IGNORE
    up = torch.rand(T, device="cuda") + 0.5
    want = reference(h, w, up, targets=y)
    (_, hv), (_, wv) = placed(h, kind), placed(w, kind)
    hb, dh = placed(torch.zeros_like(h), kind)
    wb, dw = placed(torch.zeros_like(w), kind)
    out = call(hv, wv, targets=y, up=up, dh=dh, dw=dw)
    check(out, want, dtype)
    # nothing around the results was written
    dh.fill_(9.0)
    dw.fill_(9.0)
    assert bool((hb == 9.0).all()) and bool((wb == 9.0).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_broadcast_states(dtype):
    h, w, y = states(1, 500, 64, dtype)
    h = h.expand(40, 64)
    y = (torch.arange(40, device="cuda", dtype=torch.int32) * 11) % 500
    up = torch.rand(40, device="cuda") + 0.5
    check(call(h, w, targets=y, up=up), reference(h, w, up, targets=y), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("op", ["xent", "distill"])
@pytest.mark.parametrize("limit", [1, 300_000])
def test_pieces_of_the_vocabulary(limit, op, dtype):
    T, V, D = 140, 1400, 72
    h, w, y = states(T, V, D, dtype)
    kw = dict(targets=y)
    if op == "distill":
        index, logits = teacher(T, V, 20)
        kw = dict(index=index, logits=logits, tau=2.0)
    up = torch.rand(T, device="cuda") + 0.5
    check(call(h, w, up=up, limit=limit, **kw), reference(h, w, up, **kw), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("op", ["xent", "distill"])
def test_blocks_of_rows(op, dtype):
    """A workspace limit under which the rows are taken about 1100 at a time, with blocks that no row reaches."""
    T, V, D = 3000, 300, 72
    h, w, y = states(T, V, D, dtype)
    kw = dict(targets=y)
    limit = 1_200_000 if dtype == torch.bfloat16 else 2_500_000
    up = torch.rand(T, device="cuda") + 0.5
    for ignored in (slice(5, 9), slice(700, 3000)):
        if op == "distill":
            index, logits = teacher(T, V, 20)
            index[ignored] = -1
            kw = dict(index=index, logits=logits, tau=2.0)
        else:
            kw = dict(targets=y.clone())
            kw["targets"][ignored] = IGNORE
        check(call(h, w, up=up, limit=limit, **kw), reference(h, w, up, **kw), dtype)
        check(call(h, w, up=up[:1], mean=True, limit=limit, **kw), reference(h, w, up[:1], mean=True, **kw), dtype, True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("op", ["xent", "distill"])
@pytest.mark.parametrize("mean", [False, True])
def test_gradients_from_a_kept_lse(op, dtype, mean):
    T, V, D = 140, 900, 72
    h, w, y = states(T, V, D, dtype)
    y[3] = IGNORE
    kw = dict(targets=y)
    if op == "distill":
        index, logits = teacher(T, V, 20)
        kw = dict(index=index, logits=logits, tau=2.0)
    up = torch.rand(1 if mean else T, device="cuda") + 0.5
    first = call(h, w, mean=mean, dh=None, dw=None, **kw)
    want = reference(h, w, up, mean=mean, **kw)
    check(first, want, dtype, mean)
    check(call(h, w, mean=mean, up=up, lse_in=first["lse"], **kw), want, dtype, mean)
    check(call(h, w, mean=mean, up=up, lse_in=first["lse"], dh=None, **kw), want, dtype, mean)
    check(call(h, w, mean=mean, up=up, lse_in=first["lse"], dw=None, **kw), want, dtype, mean)
    check(call(h, w, mean=mean, up=up, dw=None, **kw), want, dtype, mean)
    check(call(h, w, mean=mean, up=up, dh=None, **kw), want, dtype, mean)


@pytest.mark.parametrize("dtype", DTYPES)
def test_without_an_upstream_gradient_it_is_one(dtype):
    h, w, y = states(50, 300, 64, dtype)
    check(call(h, w, targets=y), reference(h, w, torch.ones(50, device="cuda"), targets=y), dtype)
    check(call(h, w, targets=y, mean=True), reference(h, w, torch.ones(1, device="cuda"), targets=y, mean=True), dtype,
          True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_logit_scale(dtype):
    h, w, y = states(50, 300, 64, dtype)
    up = torch.ones(50, device="cuda")
    check(call(h, w, targets=y, up=up, scale=0.125), reference(h, w, up, targets=y, scale=0.125), dtype)


@pytest.mark.parametrize("grads", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_small_losses_keep_their_digits(dtype, grads):
    """Losses of about 0.008 between logits of 60 and 55: a difference of two
    rounded values of 60 (86 in base 2) would be off by up to 2^-18; the sum of the
    exponentials, near one, is off by a few 2^-24, and a relative 2^-17 of the
    logits by 2^-17 of the loss."""
    T, V, D = 8, 500, 1024
    h, w, y = states(T, V, D, dtype)
    rows = w[y.long()].float()
    near = (y.long() + 1) % V
    w[near] = (0.92 * rows).to(dtype)
    w[y.long()] = rows.to(dtype)
    h = (60 * rows / rows.square().sum(1, keepdim=True)).to(dtype)
    up = torch.ones(T, device="cuda")
    out = call(h, w, targets=y, up=up if grads else None, dh="new" if grads else None, dw="new" if grads else None)
    want = reference(h, w, up, targets=y)[0]
    assert 1e-3 < float(want.min()) and float(want.max()) < 0.1
    assert float((out["loss"].double() - want).abs().max()) <= 16 * 2.0 ** -24


def test_extreme_logits():
    """Logits in the thousands: the softmax is one word or the other, and nothing overflows."""
    for dtype in DTYPES:
        h, w, y = states(40, 700, 64, dtype, scale=2000.0)
        up = torch.ones(40, device="cuda")
        out = call(h, w, targets=y, up=up)
        loss, lse, dh, dw, rows, top = reference(h, w, up, targets=y)
        assert top > 3000
        assert float((out["loss"].double() - loss).abs().max()) <= 1e-5 * (1 + top)
        assert float((out["lse"].double() - lse).abs().max()) <= 1e-5 * (1 + top)
        assert bool(torch.isfinite(out["dh"]).all()) and bool(torch.isfinite(out["dw"]).all())


def test_float32_magnitudes():
    """The f16 planes follow the matrices' magnitudes: tiny and huge ones lose nothing."""
    for hs, ws in ((1e-12, 1e12), (1e15, 1e-15), (1.0, 1e-30), (1e-38, 1e30)):
        h, w, y = states(40, 300, 64, torch.float32)
        h, w = h * hs, w * ws
        scale = 1.0 / (hs * ws) if hs * ws > 1e-20 else 1.0
        up = torch.ones(40, device="cuda")
        out = call(h, w, targets=y, up=up, scale=scale)
        want = reference(h, w, up, targets=y, scale=scale)
        check({k: v for k, v in out.items() if k in ("loss", "lse")}, want, torch.float32)
        for name, expect in (("dh", want[2]), ("dw", want[3])):
            if 1e-30 < float(expect.abs().max()) < 1e30:
                assert frobenius(out[name], expect) <= 2e-5 * (1 + want[5] / 4), name


def test_infinite_and_nan_states_stay_in_their_rows():
    h, w, y = states(30, 300, 64, torch.bfloat16)
    clean = call(h, w, targets=y, dw=None)
    h = h.clone()
    h[4, 3] = math.nan
    h[9, 5] = math.inf
    out = call(h, w, targets=y, dw=None)
    bad = torch.zeros(30, dtype=torch.bool, device="cuda")
    bad[4] = bad[9] = True
    assert bool(out["loss"][bad].isnan().all())
    for name in ("loss", "lse", "dh"):
        assert torch.equal(out[name][~bad], clean[name][~bad])


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_same_call_gives_the_same_bits(dtype):
    h, w, _ = states(300, 1500, 200, dtype)
    index, logits = teacher(300, 1500, 30)
    a = call(h, w, index=index, logits=logits, tau=2.0)
    for _ in range(2):
        b = call(h, w, index=index, logits=logits, tau=2.0)
        for name in a:
            assert torch.equal(a[name], b[name]), name


def test_on_another_stream():
    """Inputs made, and results read, on the stream that the call is given."""
    h, w, y = states(200, 900, 128, torch.bfloat16)
    up = torch.ones(200, device="cuda")
    want = reference(h, w, up, targets=y)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        late = torch.zeros_like(h)
        for _ in range(50):
            late.add_(1.0)
        late.copy_(h)
        out = call(late, w, targets=y, up=up, stream=side.cuda_stream)
        copies = {k: v.clone() for k, v in out.items()}
    side.synchronize()
    check(copies, want, torch.bfloat16)


def test_gradients_against_differences():
    """Central differences of the kernels' own Float32 loss along random directions.  With a step of
    0.02 the quotient's error is that of the loss, 1e-5 (1 + max |s|) over the step, and the third
    derivative's 0.02^2 / 6 of a directional derivative of unit-order curvature."""
    T, V, D = 12, 200, 48
    h, w, y = states(T, V, D, torch.float32)
    index, logits = teacher(T, V, 9)
    for kw in (dict(targets=y), dict(index=index, logits=logits, tau=1.5)):
        up = torch.rand(T, device="cuda") + 0.5
        out = call(h, w, up=up, **kw)
        top = reference(h, w, up, **kw)[5]
        for seed in range(4):
            g = torch.Generator().manual_seed(seed)
            a, b = torch.randn(T, D, generator=g).cuda(), torch.randn(V, D, generator=g).cuda()
            a, b = a / a.norm(), b / b.norm()
            step = 0.02

            def total(e):
                return float((call(h + e * a, w + e * b, dh=None, dw=None, **kw)["loss"].double() * up).sum())

            slope = (total(step) - total(-step)) / (2 * step)
            given = float((out["dh"].double() * a).sum() + (out["dw"].double() * b).sum())
            assert abs(slope - given) <= 1e-5 * (1 + top) * T / step + step ** 2 * T


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_walks_keep_their_precision(dtype):
    """A vocabulary of 70000 is summed for dh, 5000 rows for dw."""
    T, V, D = 5000, 70000, 64
    h, w, y = states(T, V, D, dtype)
    up = torch.ones(1, device="cuda")
    check(call(h, w, targets=y, mean=True, up=up), reference(h, w, up, targets=y, mean=True), dtype, True)


def test_the_example_learns():
    import subprocess
    import sys
    from pathlib import Path

    root = Path(__file__).resolve().parent.parent
    out = subprocess.run([sys.executable, str(root / "examples" / "train_head.py"), "--steps", "12", "--tokens", "200",
                          "--vocab", "1000", "--dim", "64"], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout + out.stderr


def test_through_the_tensor_api():
    """nn's losses on CUDA carrier tensors, autograd and the one-call form, against the raw entry points."""
    sw = pytest.importorskip("strideweave")
    import numpy as np
    from strideweave import Layout, Shape, Stride, Tensor

    from strideweave_b200 import CUDA, nn

    rng = np.random.default_rng(0)
    T, V, D = 40, 300, 48
    h = rng.standard_normal((T, D)).astype(np.float32)
    w = (rng.standard_normal((V, D)) * 0.2).astype(np.float32)
    y = rng.integers(0, V, T).astype(np.int32)
    y[3] = IGNORE

    def matrix(a):
        return Tensor(CUDA.from_numpy(a.ravel()), 0, Layout(Shape(list(a.shape)), Stride([a.shape[1], 1])))

    x, weight = matrix(h), matrix(w)
    targets = Tensor(CUDA.from_numpy(y), 0, Layout(Shape(T), Stride(1)))
    loss, dx, dw = nn.linear_cross_entropy_and_gradients(x, weight, targets)
    up = torch.ones(1, device="cuda")
    want = call(torch.from_numpy(h).cuda(), torch.from_numpy(w).cuda(), targets=torch.from_numpy(y).cuda(), mean=True,
                up=up)
    assert loss.carrier.to_numpy()[0] == want["loss"].cpu().numpy()[0]
    np.testing.assert_array_equal(dx.carrier.to_numpy(), want["dh"].cpu().numpy().ravel())
    np.testing.assert_array_equal(dw.carrier.to_numpy(), want["dw"].cpu().numpy().ravel())
    alone = nn.linear_cross_entropy(x, weight, targets)
    assert alone.carrier.to_numpy()[0] == loss.carrier.to_numpy()[0]
    with pytest.raises(ValueError, match="targets must have 40 elements"):
        nn.linear_cross_entropy(x, weight, Tensor(CUDA.from_numpy(y[:5]), 0, Layout(Shape(5), Stride(1))))
    assert sw is not None
