"""Checks of the linear head's losses at the tensor level, by name:

    python tests/linear_head_tensors.py NAME [NAME...]

A process of its own, because it stands in for the host framework where that is not installed."""

from __future__ import annotations

import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import numpy as np  # noqa: E402
import torch  # noqa: E402

from tests import host_stand_in  # noqa: E402

host_stand_in.install()

from strideweave import Layout, Shape, Stride, Tensor  # noqa: E402

from strideweave_b200 import CUDA, BFloat16, nn  # noqa: E402
from strideweave_b200._host import DType  # noqa: E402
from tests.test_gpu_linear_head import IGNORE, call, frobenius, reference, states, teacher  # noqa: E402

T, V, D, K = 40, 300, 48, 9
DTYPES = {torch.float32: DType.Float32, torch.bfloat16: BFloat16}


def tensor(t, requires_grad=False):
    """A torch tensor's values as a tensor of this package's carrier, in the same placement."""
    flat = t.as_strided((sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1,), (1,))
    dtype = DType.Int32 if t.dtype == torch.int32 else DTYPES[t.dtype]
    host = flat.cpu() if t.dtype == torch.int32 else flat.float().cpu()
    layout = Layout(Shape(list(t.shape)), Stride(list(t.stride()))) if t.dim() > 1 else Layout(Shape(t.shape[0]),
                                                                                              Stride(t.stride()[0]))
    return Tensor(CUDA.from_numpy(host.numpy(), dtype=dtype), 0, layout, requires_grad=requires_grad)


def values(t):
    layout = t.layout
    flat = torch.from_numpy(np.array(t.carrier.to_numpy())).cuda()
    return flat.as_strided(tuple(layout.shape.top_level), tuple(layout.stride.top_level))


def cases(placements=("rows", "columns")):
    for dtype in DTYPES:
        h0, w0, y = states(T, V, D, dtype)
        y[3] = IGNORE
        index, logits = teacher(T, V, K)
        for placement in placements:
            h, w = h0, w0
            if placement == "columns":
                h, w = h.t().contiguous().t(), w.t().contiguous().t()
            if placement == "one row":
                h = h[:1].expand(T, D)
            for op in ("xent", "distill"):
                kw = dict(targets=y) if op == "xent" else dict(index=index, logits=logits, tau=2.0)
                yield dtype, h, w, op, kw


def loss_of(op, x, weight, kw, reduction, module=False):
    if op == "xent":
        f = nn.LinearCrossEntropy(reduction=reduction) if module else nn.linear_cross_entropy
        more = {} if module else dict(reduction=reduction)
        return f(x, weight, tensor(kw["targets"]), **more)
    f = nn.LinearDistillation(temperature=2.0, reduction=reduction) if module else nn.linear_distillation
    more = {} if module else dict(reduction=reduction, temperature=2.0)
    return f(x, weight, tensor(kw["index"]), tensor(kw["logits"]), **more)


def near(got, want, dtype):
    assert frobenius(got, want) <= (5e-3 if dtype == torch.bfloat16 else 1e-4), frobenius(got, want)


def autograd():
    """loss.backward() for the mean, and for a loss per row with a gradient per row."""
    for dtype, h, w, op, kw in cases(("rows", "columns", "one row")):
        for reduction in ("mean", "none"):
            for module in (False, True):
                x, weight = tensor(h, True), tensor(w, True)
                loss = loss_of(op, x, weight, kw, reduction, module)
                if reduction == "mean":
                    up = torch.ones(1, device="cuda")
                    loss.backward()
                else:
                    up = torch.rand(T, device="cuda") + 0.5
                    loss.backward(tensor(up))
                want = reference(h, w, up, mean=reduction == "mean", **kw)
                rows = want[0].sum() / want[4].sum() if reduction == "mean" else want[0]
                assert float((values(loss).double() - rows).abs().max()) <= 4e-5 * (1 + want[5])
                near(values(x.grad), want[2], dtype)
                near(values(weight.grad), want[3], dtype)


def one_call():
    for dtype, h, w, op, kw in cases(("rows", "columns", "one row")):
        x, weight = tensor(h), tensor(w)
        for reduction in ("mean", "none"):
            if op == "xent":
                loss, dx, dw = nn.linear_cross_entropy_and_gradients(x, weight, tensor(kw["targets"]),
                                                                     reduction=reduction)
            else:
                loss, dx, dw = nn.linear_distillation_and_gradients(x, weight, tensor(kw["index"]),
                                                                    tensor(kw["logits"]), temperature=2.0,
                                                                    reduction=reduction)
            raw = call(h, w, mean=reduction == "mean", **kw)
            assert torch.equal(values(loss), raw["loss"])
            assert torch.equal(values(dx).to(dtype), raw["dh"]) and torch.equal(values(dw).to(dtype), raw["dw"])


def upstream_placements():
    """A gradient per row at another stride, behind an offset, or the same for every row."""
    for dtype, h, w, op, kw in cases(("rows",)):
        base = torch.rand(3 * T, device="cuda") + 0.5
        for up in (base[::3], base[1:2].expand(T), base[5:5 + T]):
            x, weight = tensor(h, True), tensor(w, True)
            loss = loss_of(op, x, weight, kw, "none")
            gradient = tensor(base)
            gradient.offset, gradient.layout = up.storage_offset(), Layout(Shape(T), Stride(up.stride()[0]))
            loss.backward(gradient)
            want = reference(h, w, up, **kw)
            near(values(x.grad), want[2], dtype)
            near(values(weight.grad), want[3], dtype)


def refused(error, match, f):
    try:
        f()
    except error as e:
        assert match in str(e), e
        return
    raise AssertionError(f"not refused: {match}")


def teacher_shapes():
    """Logits of as many elements as the index, in other rows."""
    for dtype, h, w, op, kw in cases(("rows",)):
        if op != "distill":
            continue
        x, weight, index = tensor(h), tensor(w), tensor(kw["index"])
        flat = kw["logits"].reshape(-1)
        for logits in (flat.reshape(K, T), flat.reshape(1, T * K)):
            refused(ValueError, "entries a row", lambda: nn.linear_distillation(x, weight, index, tensor(logits)))
        refused(ValueError, "two-mode layout", lambda: nn.linear_distillation(x, weight, index, tensor(flat)))
        refused(ValueError, "index must have", lambda: nn.linear_distillation(x, weight, tensor(kw["index"][:5]),
                                                                              tensor(kw["logits"])))


def devices():
    """A carrier that says it is on another device is refused before anything is launched."""

    def elsewhere(t):
        t.carrier._device = 1
        return t

    for dtype, h, w, op, kw in cases(("rows",)):
        x, weight = tensor(h), tensor(w)
        refused(ValueError, "weight is on device 1", lambda: loss_of(op, x, elsewhere(tensor(w)), kw, "mean"))
        if op == "xent":
            refused(ValueError, "targets is on device 1",
                    lambda: nn.linear_cross_entropy(x, weight, elsewhere(tensor(kw["targets"]))))
        else:
            for bad in ("index", "logits"):
                two = {n: elsewhere(tensor(kw[n])) if n == bad else tensor(kw[n]) for n in ("index", "logits")}
                refused(ValueError, f"{bad} is on device 1", lambda: nn.linear_distillation(x, weight, **two))
        loss = loss_of(op, x, weight, kw, "none")
        refused(ValueError, "gradient is on device 1",
                lambda: loss.backward(elsewhere(tensor(torch.ones(T, device="cuda")))))
        refused(ValueError, "gradient is on device 1",
                lambda: loss.backward(elsewhere(tensor(torch.ones(2 * T, device="cuda")[::2]))))


if __name__ == "__main__":
    for name in sys.argv[1:]:
        globals()[name]()
