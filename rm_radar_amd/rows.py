"""Device rows behind the detector: a cache of features held in 8 bits and a linear layer (include/rmr.h, "rows of features").

Operands are torch tensors on the GPU (float16, bfloat16 or float32, the last dimension packed, rows at any pitch and alignment);
work is enqueued on torch's current stream of that device and nothing is waited for, so calls can be captured into a
``torch.cuda.CUDAGraph``.  Outputs and workspaces come from torch's allocator.  Nothing is recorded for autograd.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from ._lib import InvalidArgument, check, lib

_FORMATS = {"f16": 0, "bf16": 1, "mx8": 2}
_ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "sigmoid": 4}
_types: dict = {}


def _torch():
    import torch
    if not _types:
        _types.update({torch.float16: 0, torch.bfloat16: 1, torch.float32: 2})
    return torch


def _refuse(msg):
    raise InvalidArgument(_lib.ERR_INVALID_ARGUMENT, msg)


def _stream(torch, device):
    """The raw stream torch works on (as an address: no Stream object per call where torch offers that)."""
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw(device) if raw is not None else torch.cuda.current_stream(device).cuda_stream


def _rows(t, what, width, device):
    """A tensor [..., width] as (address, type, row pitch in elements, rows)."""
    kind = _types.get(t.dtype)
    if kind is None:
        _refuse(f"{what}: dtype {t.dtype} is not float16, bfloat16 or float32")
    if t.get_device() != device:
        _refuse(f"{what} is on {t.device}, not on GPU {device}")
    if t.dim() != 2:
        if t.dim() == 0 or t.shape[-1] != width:
            _refuse(f"{what} has shape {tuple(t.shape)}, its last dimension must be {width}")
        try:
            t = t.view(-1, width) if t.numel() else t.reshape(0, width)
        except RuntimeError:
            _refuse(f"{what}: the rows of shape {tuple(t.shape)} with strides {t.stride()} are not evenly spaced")
    rows, w = t.shape
    if w != width:
        _refuse(f"{what} has rows of {w} values, not {width}")
    pitch, step = t.stride()
    if step != 1 and w > 1 and rows:
        _refuse(f"{what}: the values of a row must be packed (strides {t.stride()})")
    return t.data_ptr(), kind, pitch, rows


def _slots(torch, t, device):
    if t.dtype is not torch.int64 or t.dim() != 1 or not t.is_contiguous():
        _refuse("slots must be a packed one-dimensional int64 tensor")
    if t.get_device() != device:
        _refuse(f"slots are on {t.device}, not on GPU {device}")
    return t.data_ptr(), t.shape[0]


def _output(like, shape, width, dtype, out, device):
    """The caller's `out` or a new tensor [*shape, width] beside `like`: (tensor, address, type, row pitch, rows)."""
    if out is None:
        kind = _types.get(dtype)
        if kind is None:
            _refuse(f"dtype {dtype} is not float16, bfloat16 or float32")
        out = like.new_empty((*shape, width), dtype=dtype)
        return out, out.data_ptr(), kind, width, None
    if dtype is not None and out.dtype != dtype:
        _refuse(f"out has dtype {out.dtype}, asked for {dtype}")
    return (out, *_rows(out, "out", width, device))


class FeatureCache:
    """``slots`` rows of ``width`` values in 8 bits: per block of 32 values one power of two and 32 e4m3 values, off by at most half
    an e4m3 step of the block's largest.  A new cache holds zeros."""

    def __init__(self, slots, width, device=0):
        self._h, self._lib = C.c_void_p(), lib()
        check(self._lib.rmr_feature_cache_create(device, slots, width, C.byref(self._h)))
        self.slots, self.width, self.device = slots, width, device

    def close(self):
        if getattr(self, "_h", None) and _lib is not None and _lib._lib is not None:  # module globals are gone at interpreter exit
            _lib._lib.rmr_feature_cache_destroy(self._h)
            self._h = None

    __del__ = close

    def nbytes(self) -> int:
        """Device memory held."""
        return self._lib.rmr_feature_cache_bytes(self._h)

    def write(self, x, slots):
        """Row i of x [n, width] enters slot slots[i] (int64 [n] on the GPU).  Rows whose slot does not exist are left out; of
        rows that name one slot the last stays."""
        torch = _torch()
        p, kind, ld, n = _rows(x, "x", self.width, self.device)
        sp, m = _slots(torch, slots, self.device)
        if n != m:
            _refuse(f"{n} rows and {m} slots")
        check(self._lib.rmr_feature_cache_write(self._h, p, kind, ld, sp, n, _stream(torch, self.device)))

    def read(self, slots, dtype=None, out=None):
        """The rows in ``slots`` as [n, width] of ``dtype`` (float16 by default) or into ``out``; zeros for slots that do not exist."""
        torch = _torch()
        sp, n = _slots(torch, slots, self.device)
        out, p, kind, ld, m = _output(slots, (n,), self.width, dtype or (torch.float16 if out is None else None), out, self.device)
        if m is not None and n != m:
            _refuse(f"{n} slots and {m} rows of out")
        check(self._lib.rmr_feature_cache_read(self._h, sp, n, p, kind, ld, _stream(torch, self.device)))
        return out


class Linear:
    """``act(x W^T + bias) + residual``, accumulated in f32 and rounded once.

    weight: [out_features, in_features], torch tensor (GPU or host) or numpy array; bias: [out_features] or None.  ``format``: "f16"
    / "bf16" (x and W of that type) or "mx8" (x and W in blocks of 8-bit values as a FeatureCache holds them; x of any type is
    quantised within the call).  Weights of other types than float16, bfloat16 and float32 are rounded to float32 first.

    An "mx8" layer's 16-bit results come from products cut 13 bits below the largest of their group: sums are about 1.5e-5 of
    the norm of their products off, which shows where they cancel to a few per cent of it.  Float32 results (``out_dtype``) are summed
    in full float32, at half the rate.

    ``activation``: none, relu, silu, gelu (v / 2 erfc(-v / sqrt 2)), sigmoid."""

    def __init__(self, weight, bias=None, activation="none", format="f16", device=None):
        torch = _torch()
        if format not in _FORMATS:
            _refuse(f"format {format!r} is none of {sorted(_FORMATS)}")
        if activation not in _ACTIVATIONS:
            _refuse(f"activation {activation!r} is none of {sorted(_ACTIVATIONS)}")
        w = torch.as_tensor(weight)
        if w.dim() != 2:
            _refuse(f"weight has shape {tuple(w.shape)}, not [out_features, in_features]")
        if w.dtype not in _types:
            w = w.float()
        if device is None:
            device = w.device.index if w.device.type == "cuda" else 0
        elif w.device.type == "cuda" and w.device.index != device:
            _refuse(f"weight is on {w.device}, not on GPU {device}")
        if w.stride(1) != 1 or (w.shape[0] > 1 and w.stride(0) < w.shape[1]):
            w = w.contiguous()
        b = None
        if bias is not None:
            b = torch.as_tensor(bias)
            if b.shape != (w.shape[0],):
                _refuse(f"bias has shape {tuple(b.shape)}, not ({w.shape[0]},)")
            b = b.to(device=w.device, dtype=torch.float32).contiguous()
        cfg = _lib.LinearCfg(device, w.shape[1], w.shape[0], _FORMATS[format], _ACTIVATIONS[activation])
        on_gpu = w.device.type == "cuda"
        stream = torch.cuda.current_stream(device).cuda_stream if on_gpu else None
        self._h, self._lib = C.c_void_p(), lib()
        check(self._lib.rmr_linear_create(C.byref(cfg), w.data_ptr(), _types[w.dtype], w.stride(0), b.data_ptr() if b is not None else None,
                                      _lib.MEM_DEVICE if on_gpu else _lib.MEM_HOST, stream, C.byref(self._h)))
        self.in_features, self.out_features, self.device = w.shape[1], w.shape[0], device
        self.format, self.activation = format, activation

    def close(self):
        if getattr(self, "_h", None) and _lib is not None and _lib._lib is not None:  # module globals are gone at interpreter exit
            _lib._lib.rmr_linear_destroy(self._h)
            self._h = None

    __del__ = close

    def _run(self, torch, like, x, x_kind, ldx, rows, lead, residual, out, out_dtype, cache, slots):
        out, p, kind, ldy, n = _output(like, lead, self.out_features, out_dtype, out, self.device)
        if n is not None and n != rows:
            _refuse(f"out has {n} rows, the call {rows}")
        r, ldr = None, 0
        if residual is not None:
            r, r_kind, ldr, n = _rows(residual, "residual", self.out_features, self.device)
            if n != rows or r_kind != kind:
                _refuse(f"residual has {n} rows of {residual.dtype}, the output {rows} of {out.dtype}")
        call = _lib.LinearCall(x, x_kind, ldx, rows, r, ldr, p, kind, ldy)
        at = C.byref(call)
        if rows > _lib.LINEAR_FEW_ROWS:
            need = C.c_size_t()
            check(self._lib.rmr_linear_workspace(self._h, at, cache is not None, C.byref(need)))
            if need.value:
                space = out.new_empty(need.value, dtype=torch.uint8)
                call.workspace, call.workspace_bytes = space.data_ptr(), need.value
        stream = _stream(torch, self.device)
        if cache is None:
            check(self._lib.rmr_linear_run(self._h, at, stream))
        else:
            check(self._lib.rmr_linear_run_kept(self._h, cache, slots, at, stream))
        return out

    def __call__(self, x, residual=None, out=None, out_dtype=None):
        """x [..., in_features] -> [..., out_features] of ``out_dtype`` (x's by default), or into ``out``.  ``residual``: like the
        output, may be ``out`` itself."""
        torch = _torch()
        p, kind, ld, n = _rows(x, "x", self.in_features, self.device)
        return self._run(torch, x, p, kind, ld, n, x.shape[:-1], residual, out, out_dtype or (x.dtype if out is None else None), None, None)

    def kept(self, cache, slots, residual=None, out=None, out_dtype=None):
        """The layer on the rows that ``cache`` holds in ``slots`` (int64 [n] on the GPU): [n, out_features] of ``out_dtype`` (float16 by
        default).  "mx8" layers only."""
        torch = _torch()
        sp, n = _slots(torch, slots, self.device)
        return self._run(torch, slots, None, 0, 0, n, (n,), residual, out, out_dtype or (torch.float16 if out is None else None), cache._h, sp)
