"""Device storage and strided views for the matmul hot path.

Mirrors the reference's host tensor model for device memory:
  * `DeviceBuffer` ~ BufferHandle::Device{device_ordinal, address, bytes}
    (src/momiru/tensor_light/execution/runtime.rs:297-301), plus an allocation
    identity so the binder can prove an output disjoint from its inputs.
  * `DeviceView` ~ Shape{dims, strides} over a storage with a base offset
    (tensor/shape.rs:130-206, TensorStoragePlan plan.rs:1285-1307), with the
    zero-copy view operations `transpose`, `narrow`, `slice` and
    `as_strided_view` of TensorView (tensor/view.rs:450, 791, 800, 488).
Device memory is allocated through torch (plumbing only); compute never goes
through torch.
"""
from __future__ import annotations

import enum
import itertools
from dataclasses import dataclass, field, replace

import numpy as np

from . import _abi

_alloc_ids = itertools.count(1)


class ViewError(ValueError):
    pass


class DType(enum.Enum):
    """Element types of a view: f32 everywhere, the others where an operator takes them."""
    F32 = (0, 4, "float32")
    BF16 = (1, 2, "bfloat16")
    F16 = (2, 2, "float16")
    I32 = (3, 4, "int32")

    @property
    def code(self) -> int:
        """The ABI's MMR_DTYPE_* value."""
        return self.value[0]

    @property
    def itemsize(self) -> int:
        return self.value[1]

    @property
    def torch(self):
        import torch
        return getattr(torch, self.value[2])

    @staticmethod
    def of_torch(dtype) -> "DType":
        for d in DType:
            if str(dtype) == f"torch.{d.value[2]}":
                return d
        raise ViewError(f"element type {dtype} is not one of {', '.join(d.name for d in DType)}")


@dataclass
class DeviceBuffer:
    """A device allocation (or a raw external handle) the caller owns."""
    address: int
    bytes: int
    device_ordinal: int = 0
    allocation_id: int = field(default_factory=lambda: next(_alloc_ids))
    owner: object = None  # keeps a torch tensor alive when we allocated it

    @staticmethod
    def allocate(nbytes: int, device_ordinal: int = 0) -> "DeviceBuffer":
        import torch
        n = max(1, (nbytes + 3) // 4)
        t = torch.empty(n, dtype=torch.float32, device=f"cuda:{device_ordinal}")
        return DeviceBuffer(t.data_ptr(), n * 4, device_ordinal, owner=t)

    @staticmethod
    def from_torch(t) -> "DeviceBuffer":
        """Borrow the storage of a CUDA torch tensor (no copy)."""
        st = t.untyped_storage()
        return DeviceBuffer(st.data_ptr(), st.nbytes(), t.device.index or 0, owner=t)


@dataclass(frozen=True)
class DeviceView:
    buffer: DeviceBuffer
    dims: tuple
    strides: tuple          # element strides (signed)
    offset: int = 0         # element offset of [0, .., 0]
    dtype: DType = DType.F32

    # ---------------------------------------------------------------- create
    @staticmethod
    def contiguous(buffer: DeviceBuffer, dims, offset: int = 0, dtype: DType = DType.F32) -> "DeviceView":
        dims = tuple(int(d) for d in dims)
        strides, acc = [], 1
        for d in reversed(dims):
            strides.append(acc)
            acc *= max(d, 1)
        return DeviceView(buffer, dims, tuple(reversed(strides)), offset, dtype)

    @staticmethod
    def empty(dims, device_ordinal: int = 0, dtype: DType = DType.F32) -> "DeviceView":
        n = int(np.prod(dims)) if len(dims) else 1
        return DeviceView.contiguous(DeviceBuffer.allocate(dtype.itemsize * n, device_ordinal), dims, dtype=dtype)

    @staticmethod
    def from_torch(t) -> "DeviceView":
        """The CUDA tensor's own elements as a view (no copy); it keeps the tensor alive."""
        return DeviceView(DeviceBuffer.from_torch(t), tuple(t.shape), tuple(t.stride()), t.storage_offset(),
                          DType.of_torch(t.dtype))

    @staticmethod
    def from_host(arr: np.ndarray, device_ordinal: int = 0) -> "DeviceView":
        import torch
        a = np.ascontiguousarray(arr, dtype=np.float32)
        t = torch.from_numpy(a).to(f"cuda:{device_ordinal}")
        return DeviceView.contiguous(DeviceBuffer.from_torch(t), a.shape)

    # ------------------------------------------------------------ properties
    @property
    def rank(self) -> int:
        return len(self.dims)

    @property
    def numel(self) -> int:
        return int(np.prod(self.dims)) if self.dims else 1

    def is_row_major_contiguous(self) -> bool:
        return self == DeviceView.contiguous(self.buffer, self.dims, self.offset, self.dtype)

    # ------------------------------------------------------------ view ops
    def transpose(self, a: int = -2, b: int = -1) -> "DeviceView":
        a %= self.rank
        b %= self.rank
        d, s = list(self.dims), list(self.strides)
        d[a], d[b] = d[b], d[a]
        s[a], s[b] = s[b], s[a]
        return replace(self, dims=tuple(d), strides=tuple(s))

    def narrow(self, axis: int, start: int, length: int) -> "DeviceView":
        axis %= self.rank
        if start < 0 or length < 0 or start + length > self.dims[axis]:
            raise ViewError(f"narrow({axis}, {start}, {length}) outside extent {self.dims[axis]}")
        d = list(self.dims)
        d[axis] = length
        return replace(self, dims=tuple(d), offset=self.offset + start * self.strides[axis])

    def slice(self, specs) -> "DeviceView":
        """specs: one (start, stop, step>0) tuple or None (full axis) per axis."""
        d, s, off = list(self.dims), list(self.strides), self.offset
        for ax, spec in enumerate(specs):
            if spec is None:
                continue
            start, stop, step = spec
            if step <= 0 or not (0 <= start <= stop <= self.dims[ax]):
                raise ViewError(f"slice spec {spec} invalid for axis {ax}")
            off += start * s[ax]
            d[ax] = (stop - start + step - 1) // step
            s[ax] *= step
        return replace(self, dims=tuple(d), strides=tuple(s), offset=off)

    def as_strided_view(self, dims, strides, offset: int | None = None) -> "DeviceView":
        return replace(self, dims=tuple(dims), strides=tuple(strides), offset=self.offset if offset is None else offset)

    def unsqueeze(self, axis: int) -> "DeviceView":
        d, s = list(self.dims), list(self.strides)
        d.insert(axis, 1)
        s.insert(axis, 0)
        return replace(self, dims=tuple(d), strides=tuple(s))

    # ----------------------------------------------------------- host copies
    def torch_view(self):
        """A torch view over the same memory (for copies in and out)."""
        import torch
        base = self.buffer.owner
        if base is None or not isinstance(base, torch.Tensor):
            raise ViewError("buffer not allocated through torch")
        if base.dtype != self.dtype.torch:
            if self.dtype == DType.F32:
                raise ViewError("buffer not allocated through torch as f32")
            # DeviceBuffer.allocate counts f32 words: the same bytes as this type
            flat = torch.as_strided(base, (base.untyped_storage().nbytes() // base.element_size(),), (1,), 0)
            base = flat.view(self.dtype.torch)
        # as_strided offsets are absolute within the storage, as ours are.
        return torch.as_strided(base, self.dims, self.strides, self.offset)

    def to_host(self) -> np.ndarray:
        t = self.torch_view().cpu()
        return (t.float() if self.dtype == DType.BF16 else t).numpy()

    def copy_from_host(self, arr: np.ndarray) -> None:
        import torch
        host = np.int32 if self.dtype == DType.I32 else np.float32  # f32 holds no integer past 2^24
        self.torch_view().copy_(torch.from_numpy(np.ascontiguousarray(arr, dtype=host)))

    # ------------------------------------------------------------------ ABI
    def to_abi(self) -> _abi.MmrView:
        """The view as the f32 MatMul node takes it."""
        if self.dtype != DType.F32:
            raise ViewError(f"a view of {self.dtype.name} where the MatMul node takes F32")
        return self._abi_view()

    def _abi_view(self) -> _abi.MmrView:
        if self.rank > _abi.MAX_RANK:
            raise ViewError(f"rank {self.rank} above {_abi.MAX_RANK}")
        v = _abi.MmrView()
        v.address = self.buffer.address
        v.bytes = self.buffer.bytes
        v.base_offset_bytes = self.dtype.itemsize * self.offset
        v.rank = self.rank
        v.device_ordinal = self.buffer.device_ordinal
        for i, (d, s) in enumerate(zip(self.dims, self.strides)):
            v.dims[i] = d
            v.strides[i] = s
        v.allocation_id = self.buffer.allocation_id
        return v

    def to_abi_tensor(self):
        """The view with its element type (MmrTensor of include/momiru_ops.h)."""
        from . import _ops_abi
        return _ops_abi.MmrTensor(self._abi_view(), self.dtype.code, 0)
