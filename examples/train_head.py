"""Trains a linear head over a vocabulary: distillation from a teacher's top
logits first, then cross entropy against words.

    python examples/train_head.py [--steps N] [--tokens T] [--vocab V] [--dim D]

The hidden states are fixed random features and the teacher is a random head
over them.  The student starts near zero and sees, in the first half of the
steps, the teacher's top 16 logits of each token at temperature 2, and in the
second half words drawn from the teacher's distribution, every eighth token
ignored.  The logits [T, V] are never held on the device; the losses, their
gradients and the update run there through the C ABI, without a framework on
the host side.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from strideweave_b200 import _native as N  # noqa: E402
from strideweave_b200 import kernels  # noqa: E402

IGNORE = -100
TOP = 16


def upload(a: np.ndarray) -> N.DeviceBuffer:
    buf = N.DeviceBuffer(a.nbytes)
    buf.upload(np.ascontiguousarray(a))
    return buf


def read(buf: N.DeviceBuffer) -> float:
    out = np.empty(1, np.float32)
    buf.download(out)
    return float(out[0])


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--tokens", type=int, default=512)
    ap.add_argument("--vocab", type=int, default=4000)
    ap.add_argument("--dim", type=int, default=128)
    ap.add_argument("--lr", type=float, default=20.0)
    a = ap.parse_args()
    T, V, D = a.tokens, a.vocab, a.dim
    rng = np.random.default_rng(0)

    h = rng.standard_normal((T, D), dtype=np.float32)
    teacher = (rng.standard_normal((V, D)) * (3.0 / np.sqrt(D))).astype(np.float32)
    logits = h @ teacher.T
    index = np.argsort(-logits, axis=1)[:, :TOP].astype(np.int32)
    top = np.take_along_axis(logits, index, axis=1)
    p = np.exp(logits - logits.max(axis=1, keepdims=True))
    cum = np.cumsum(p / p.sum(axis=1, keepdims=True), axis=1)
    words = np.minimum((cum < rng.random((T, 1))).sum(axis=1), V - 1).astype(np.int32)
    words[::8] = IGNORE

    d_h, d_w = upload(h), upload((rng.standard_normal((V, D)) * 0.02).astype(np.float32))
    d_index, d_top, d_words = upload(index), upload(top), upload(words)
    d_dw, d_loss = N.DeviceBuffer(V * D * 4), N.DeviceBuffer(4)
    head = ("Float32", d_h.ptr, (D, 1), d_w.ptr, (D, 1), T, V, D)

    first: dict[str, float] = {}
    for step in range(a.steps):
        if step < a.steps // 2:
            name = "distillation"
            kernels.linear_distillation(*head, d_index.ptr, d_top.ptr, TOP, temperature=2.0, reduction="mean",
                                        loss_ptr=d_loss.ptr, dw_ptr=d_dw.ptr)
        else:
            name = "cross entropy"
            kernels.linear_cross_entropy(*head, d_words.ptr, ignore_index=IGNORE, reduction="mean",
                                         loss_ptr=d_loss.ptr, dw_ptr=d_dw.ptr)
        N.check(N.lib.sw_elementwise_f32(N.SW_EW_AXPY, V * D, d_w.ptr, d_dw.ptr, d_w.ptr, -a.lr, None))
        if step % 10 == 0 or step == a.steps - 1 or name not in first:
            loss = read(d_loss)
            first.setdefault(name, loss)
            print(f"step {step:3d}  {name:13s} loss {loss:.4f}")
    N.raise_device_status()
    assert read(d_loss) < first["cross entropy"], "the loss did not fall"


if __name__ == "__main__":
    main()
