"""A small stand-in for the host framework, for tests of what this package adds at the tensor level where the
framework itself is not installed: layouts of flat modes, tensors, and a graph of one operation.  It holds only what
those tests touch, and says nothing about the framework's own behaviour; `install` leaves a real one alone."""

from __future__ import annotations

import contextlib
import sys
import types
from typing import Any


class Modes:
    def __init__(self, modes: Any) -> None:
        self.top_level = [modes] if isinstance(modes, int) else list(modes)

    def __eq__(self, other: Any) -> bool:
        return self.top_level == other.top_level


class Layout:
    def __init__(self, shape: Modes, stride: Modes) -> None:
        self.shape, self.stride = shape, stride

    def __len__(self) -> int:
        return len(self.shape.top_level)

    def __eq__(self, other: Any) -> bool:
        return self.shape == other.shape and self.stride == other.stride

    def places(self) -> list[int]:
        out = [0]
        for extent, step in zip(self.shape.top_level, self.stride.top_level):
            out = [p + i * step for p in out for i in range(extent)]
        return out

    @property
    def is_injective(self) -> bool:
        return len(set(self.places())) == len(self.places())

    @property
    def cosize(self) -> int:
        return max(self.places(), default=-1) + 1


class Tensor:
    def __init__(self, carrier: Any, offset: int, layout: Layout, requires_grad: bool = False) -> None:
        self.carrier, self.offset, self.layout, self.requires_grad = carrier, offset, layout, requires_grad
        self.grad: Any = None
        self.made_by: Any = None

    def _require_single_subtensor(self, what: str) -> None:
        pass

    def size(self) -> int:
        return len(self.layout.places())

    def backward(self, gradient: Any = None) -> None:
        if gradient is None:
            gradient = Tensor(self.carrier.new_like([1.0] * self.size()), 0, self.layout)
        for t, g in zip(self.made_by.inputs(), self.made_by.backward(gradient)):
            if t.requires_grad:
                t.grad = g


class Operation:
    def __init__(self) -> None:
        self.ctx: dict[str, Any] = {}

    def forward(self, *inputs: Any) -> Tensor:
        self.taken = inputs
        out = self._forward(*inputs)
        out.made_by = self
        return out

    def inputs(self) -> tuple:
        return self.taken


class Carrier:
    def dispatch_op(self, name: str) -> Any:
        return self._dispatch_op(name)

    def is_mutable(self) -> bool:
        return self._is_mutable()

    def _increment_version(self) -> None:
        pass


class SimpleDType:
    def __init__(self, name: str, bits: int = 0, supertype: Any = None) -> None:
        self.name = name


class DType:
    Floating = SimpleDType("Floating")

    @staticmethod
    def from_name(name: str) -> Any:
        raise KeyError(name)


for _name in ("Float32", "Float64", "Int32", "Bool", "E4M3", "E8M0", "E2M1", "MXFP8_E4M3", "MXFP4"):
    setattr(DType, _name, SimpleDType(_name))


class Capability:
    @staticmethod
    def from_plan(plan: Any) -> Any:
        return plan


def install() -> bool:
    """Makes `strideweave` importable; True where this stand-in is it."""
    try:
        import strideweave  # noqa: F401

        return False
    except ImportError:
        pass

    def ignore(*args: Any, **kw: Any) -> None:
        return None

    contents = {
        "strideweave": dict(Carrier=Carrier, Layout=Layout, Shape=Modes, Stride=Modes, Swizzle=type("Swizzle", (), {}),
                            Tensor=Tensor, no_grad=contextlib.nullcontext, CPU=type("CPU", (Carrier,), {})),
        "strideweave.carriers": {},
        "strideweave.carriers.dtype": dict(DType=DType, SimpleDType=SimpleDType),
        "strideweave.carriers.operation_capability": dict(
            OperationCapability=Capability, UnsupportedOperationPlan=type("UnsupportedOperationPlan", (Exception,), {}),
            register_operation_capabilities=ignore, require_capability=ignore),
        "strideweave.carriers.operation_helpers": dict(Operation=Operation),
        "strideweave.carriers.operation_policy": dict(resolve_operation_plan=ignore),
        "strideweave.carriers.move": dict(ElementwiseMoveOperation=Operation, MoveOperation=Operation,
                                          dispatch_move=ignore, register_move_operation=ignore),
        "strideweave.core": {},
        "strideweave.core._representation": dict(Subtensor=type("Subtensor", (), {}),
                                                 TensorRepresentation=type("TensorRepresentation", (), {})),
    }
    for name, values in contents.items():
        module = types.ModuleType(name)
        module.__dict__.update(values)
        sys.modules[name] = module
    return True
