"""Forward operators with weights laid out once (``zkml_linear_*`` of the C ABI).

* ``LinearM31``      -- y = f(x W + b) + r mod p: a Linear layer with its activation and residual;
* ``GatedLinearM31`` -- h = f(x Wg + bg) * (x Wu + bu) mod p: the up side of a gated feed-forward
  block, both projections, the activation and the product in one launch;
* ``gated_ffn_m31``  -- the two in a row: the whole gated feed-forward block.

They compute what the layer reductions of this package prove: ``keep=True`` also returns the
projections (the activation's input, and the second factor of the gated product).  Values are M31
words; x is a CUDA tensor of int32 (or uint32) on the handle's device, used in place with any row
stride, or a numpy uint32 array, which is copied and answered with numpy arrays.  Calls run on the
device's current torch stream.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional

import numpy as np

from . import ACTIVATION_TAGS, InvalidArgument, _check, context, lib


# zkml_linear_call, field for field: x, m, ldx, x_bits, activation, residual, ld_residual, out, ld_out,
# pre, ld_pre, up, ld_up, workspace, workspace_bytes, stream, pointers_checked
_CALL = struct.Struct("@PNNiiPNPNPNPNPNPi4x")


_TAGS = {None: 0, "none": 0, "relu": 1, **ACTIVATION_TAGS}
_STREAM_LEGACY = 1  # cudaStreamLegacy: torch's default stream (0) by a handle that is not NULL


def _tag(activation) -> int:
    tag = _TAGS.get(activation)
    if tag is not None:
        return tag
    if isinstance(activation, str) or activation is None:
        tag = _TAGS.get(activation.lower() if isinstance(activation, str) else None)
        if tag is None:
            raise InvalidArgument(1, f"unknown activation {activation!r}")
        return tag
    return int(activation)


def _is_tensor(x) -> bool:
    return hasattr(x, "data_ptr") and hasattr(x, "is_cuda")


_torch_module = None


def _torch():
    global _torch_module
    if _torch_module is None:
        import torch

        _torch_module = torch
    return _torch_module


_forward_fn = None


def _forward(check):
    """zkml_linear_forward (_checked) with the handle as a plain integer and the packed call as bytes."""
    global _forward_fn
    if _forward_fn is None:
        sig = C.CFUNCTYPE(C.c_int, C.c_void_p, C.c_char_p)
        _forward_fn = tuple(sig(C.cast(f, C.c_void_p).value)
                            for f in (lib().zkml_linear_forward, lib().zkml_linear_forward_checked))
    return _forward_fn[1 if check else 0]


class _Weights:
    """Shared part of the two operators: the handle, the call and its checks."""

    def __init__(self, weights, biases, device: Optional[int]):
        first = weights[0]
        if device is None:
            device = first.device.index if _is_tensor(first) and first.is_cuda else 0
        self.device = int(device)
        self._handle = None
        self._need = {}
        keep, ptrs = [], []
        for w in weights:
            if len(w.shape) != 2:
                raise InvalidArgument(1, "a weight is a matrix")
            if tuple(w.shape) != tuple(first.shape):
                raise InvalidArgument(1, "the weights of a gated block have the same shape")
        weights = [self._words(w, "weight") for w in weights]
        if any(_strides(w) != _strides(weights[0]) for w in weights):
            weights = [w.contiguous() if _is_tensor(w) else np.ascontiguousarray(w) for w in weights]
        for w in weights:
            keep.append(w)
            ptrs.append(_pointer(w))
        self.k, self.n = int(first.shape[0]), int(first.shape[1])
        for b in biases:
            if b is None:
                ptrs.append(None)
                continue
            if tuple(b.shape) != (self.n,):
                raise InvalidArgument(1, f"a bias has {self.n} values")
            b = self._words(b.contiguous() if _is_tensor(b) else np.ascontiguousarray(b), "bias")
            keep.append(b)
            ptrs.append(_pointer(b))
        self._ctx = context(self.device)
        h = C.c_void_p()
        create = lib().zkml_linear_create_gated if len(weights) == 2 else lib().zkml_linear_create
        rs, cs = _strides(weights[0])
        _check(create(self._ctx.handle, *ptrs[:len(weights)], self.k, self.n, rs, cs, *ptrs[len(weights):],
                      self._stream(), C.byref(h)))
        self._handle = h

    def close(self) -> None:
        if self._handle:
            lib().zkml_linear_destroy(self._handle)
            self._handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _stream(self) -> int:
        torch = _torch()
        if not torch.cuda.is_available():
            return 0
        return torch.cuda.current_stream(self.device).cuda_stream or _STREAM_LEGACY

    def _words(self, x, name):
        """x as words the library can read: a tensor of 32-bit integers (CUDA: on this device), or an array."""
        if not _is_tensor(x):
            x = np.asarray(x)
            if x.dtype not in (np.uint32, np.int32):
                raise InvalidArgument(1, f"{name}: M31 words are uint32 or int32")
            # the library takes addresses and strides in whole words, upwards
            whole = x.ctypes.data % x.itemsize == 0 and all(s >= 0 and s % x.itemsize == 0 for s in x.strides)
            return x if whole else np.array(x, order="C")
        torch = _torch()
        if x.dtype not in (torch.int32, torch.uint32):
            raise InvalidArgument(1, f"{name}: M31 words are int32 or uint32")
        if x.is_cuda and x.device.index != self.device:
            raise InvalidArgument(1, f"{name} is on {x.device}, the weights are on cuda:{self.device}")
        return x

    def _rows(self, x, width, name, m=None):
        """(pointer, rows, row stride) of a matrix of words on this device; one row may be 1-D."""
        if getattr(x, "is_cuda", False) and x.dtype is _torch().int32 and x.get_device() == self.device and x.dim() == 2:
            rows, cols = x.shape
            ld, one = x.stride()
            if cols == width and (one == 1 or width == 1) and rows and (m is None or rows == m):
                return x.data_ptr(), rows, ld if rows > 1 else width  # the common form, in a few attribute reads
        if not _is_tensor(x):
            raise InvalidArgument(1, f"{name}: arguments beside a tensor x are tensors on cuda:{self.device} too")
        x = self._words(x, name)
        if not x.dim() or x.shape[-1] != width:
            raise InvalidArgument(1, f"{name} has rows of {width} words")
        if width > 1 and x.stride(-1) != 1:
            raise InvalidArgument(1, f"{name}: the words of a row must be contiguous")
        lead = [(int(d), int(st)) for d, st in zip(x.shape[:-1], x.stride()[:-1]) if d != 1]
        rows, ld = 1, width
        if lead:
            ld = lead[-1][1]
            for d, st in reversed(lead):
                if st != ld * rows and d:
                    raise InvalidArgument(1, f"{name}: the rows must be at one stride")
                rows *= d
        if not x.is_cuda:
            raise InvalidArgument(1, f"{name} is not on cuda:{self.device}")
        if m is not None and rows != m:
            raise InvalidArgument(1, f"{name} has {rows} rows, x has {m}")
        return x.data_ptr(), rows, ld

    def _call(self, x, activation, residual, out, pre, up, keep, x_bits, check):
        if self._handle is None:
            raise InvalidArgument(1, "the weights were closed")
        torch = _torch()
        k, n = self.k, self.n
        xp, m, ldx = self._rows(x, k, "x")
        rp = ldr = op = ldo = pp = ldp = pu = ldu = ws = 0
        if residual is not None:
            if _is_tensor(residual) and residual.dim() == 1 and m != 1:
                residual = residual.unsqueeze(0).expand(m, n)  # one row for every token
            rp, _, ldr = self._rows(residual, n, "residual", m)
        if out is None or (keep and (pre is None or (up is None and self._gated))):
            shape = (*x.shape[:-1], n)
        if out is None:
            out = x.new_empty(shape, dtype=torch.int32)
            op, ldo = out.data_ptr(), n
        else:
            op, _, ldo = self._rows(out, n, "out", m)
        results = [out]
        if pre is not None:
            pp, _, ldp = self._rows(pre, n, "pre", m)
        elif keep:
            pre = x.new_empty(shape, dtype=torch.int32)
            pp, ldp = pre.data_ptr(), n
        if pre is not None:
            results.append(pre)
        if up is not None:
            pu, _, ldu = self._rows(up, n, "up", m)
        elif keep and self._gated:
            up = x.new_empty(shape, dtype=torch.int32)
            pu, ldu = up.data_ptr(), n
        if up is not None:
            results.append(up)
        need = self._need.get((m, x_bits))
        if need is None:
            size = C.c_size_t(0)
            _check(lib().zkml_linear_workspace(self._handle, m, int(x_bits), C.byref(size)))
            if len(self._need) > 1000:
                self._need.clear()
            need = self._need[(m, x_bits)] = size.value
        if need:
            workspace = x.new_empty(need, dtype=torch.uint8)
            ws = workspace.data_ptr()
        stream = torch._C._cuda_getCurrentRawStream(self.device) or _STREAM_LEGACY
        call = _CALL.pack(xp, m, ldx, int(x_bits), _tag(activation), rp, ldr, op, ldo, pp, ldp, pu, ldu, ws, need, stream,
                          1)
        rc = _forward(check)(self._handle.value, call)
        if rc:
            _check(rc)
        return results

    def check(self) -> None:
        """Waits for the current stream; raises if a call with check=False, on any stream, met a word >= 2^31 or
        an activation that does not fit its x_bits.  Each finding is raised once."""
        _check(lib().zkml_linear_check(self._handle, self._stream()))

    def _run(self, x, activation, residual, out, pre, up, keep, x_bits, check):
        if x.__class__ is _torch().Tensor or _is_tensor(x):
            r = self._call(x, activation, residual, out, pre, up, keep, x_bits, check)
            return r[0] if len(r) == 1 else tuple(r)
        if out is not None or pre is not None or up is not None:
            raise InvalidArgument(1, "output tensors go with a tensor x")
        r = self._call(self._upload(x, "x"), activation, None if residual is None else self._upload(residual, "residual"),
                       None, None, None, keep, x_bits, True)
        r = [t.cpu().numpy().view(np.uint32) for t in r]
        return r[0] if len(r) == 1 else tuple(r)

    def _upload(self, x, name):
        if _is_tensor(x):
            return x
        w = np.ascontiguousarray(self._words(x, name)).view(np.int32)
        return _torch().from_numpy(w).to(f"cuda:{self.device}")


def _strides(w):
    if _is_tensor(w):
        return tuple(int(s) for s in w.stride())
    w = np.asarray(w)
    return tuple(int(s) // w.itemsize for s in w.strides)


def _pointer(w) -> int:
    return w.data_ptr() if _is_tensor(w) else w.ctypes.data


class LinearM31(_Weights):
    """y = f(x W + b) + r mod p.  weight: k x n M31 words (a CUDA tensor, also transposed, or an
    array), bias: n words or None; both are copied into the kernels' layout, once."""

    _gated = False

    def __init__(self, weight, bias=None, device: Optional[int] = None):
        super().__init__([weight], [bias], device)

    def __call__(self, x, activation=None, residual=None, out=None, pre=None, keep: bool = False, x_bits: int = 31,
                 check: bool = True):
        """x: (..., k), of at least one row; returns y (..., n), or (y, x W + b) with keep (or a tensor for pre).

        activation: None, "relu", "gelu", "sigmoid", "softmax", "silu" or a type tag; residual: as y, or
        one row of n words for all; out / pre: int32 tensors to write, of any row stride (out may be the
        residual); x_bits: the width x is quantised to (8, 16, or 31 for any field element).
        check=True waits for the call and raises InvalidArgument for a word >= 2^31 or an x outside
        x_bits in this call; check=False returns at once (and can be captured into a CUDA graph), and
        check() reports later."""
        return self._run(x, activation, residual, out, pre, None, keep, x_bits, check)


class GatedLinearM31(_Weights):
    """h = f(x Wg + bg) * (x Wu + bu) mod p; weights and biases as LinearM31's."""

    _gated = True

    def __init__(self, w_gate, w_up, bias_gate=None, bias_up=None, device: Optional[int] = None):
        super().__init__([w_gate, w_up], [bias_gate, bias_up], device)

    def __call__(self, x, activation="silu", out=None, gate=None, up=None, keep: bool = False, x_bits: int = 31,
                 check: bool = True):
        """x: (..., k); returns h (..., n), or (h, x Wg + bg, x Wu + bu) with keep; the rest as
        LinearM31's call."""
        return self._run(x, activation, None, out, gate, up, keep, x_bits, check)


def gated_ffn_m31(x, gated: GatedLinearM31, down: LinearM31, activation="silu", residual=None, x_bits: int = 31,
                  check: bool = True):
    """A gated feed-forward block: (f(x Wg + bg) * (x Wu + bu)) Wd + bd + r mod p.  h is a full field
    element, so the down projection takes it as one, whatever x_bits."""
    h = gated(x, activation=activation, x_bits=x_bits, check=check)
    return down(h, residual=residual, x_bits=31, check=check)
