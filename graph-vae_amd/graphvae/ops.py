"""Group norm with an activation, 8-bit activation checkpoints and the gradients that read them.

Operators on node features laid out (graphs, rows, channels), channels last, on the current HIP
stream of the current device (libgvae_hip.so; there is no CPU fallback):

  group_norm_act            forward, optionally leaving 8-bit checkpoints of its input and output
  group_norm_act_backward   gradients, from the input or from its checkpoint
  checkpoint8               an activation into an 8-bit checkpoint; Checkpoint8.read() brings it back
  linear_wgrad8             weight and bias gradient of a linear layer from its input's checkpoint

They are plain calls: nothing here is recorded by autograd, and a tensor that requires grad is refused while
grad mode is on (a graph would end there without a word).  Call them under `torch.no_grad()` or from the
forward and backward of a `torch.autograd.Function`.  `GraphVAE(norm="group")` builds its encoder from the same
kernels, and its backward from the gradients here.
"""
from __future__ import annotations

from ctypes import c_float, c_int, c_int64, c_void_p
from typing import NamedTuple

import torch

from . import _hip

_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACT = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}
BLOCK = 32

_bound = None


def _bind():
    global _bound
    if _bound is None:
        L = _hip.lib()
        L.gvae_ckpt8_write.argtypes = [c_void_p, c_int, c_int64, c_int, c_int64, c_void_p, c_void_p, c_void_p]
        L.gvae_ckpt8_read.argtypes = [c_void_p, c_void_p, c_int64, c_int, c_void_p, c_int, c_int64, c_void_p]
        L.gvae_group_norm_ws_bytes.argtypes = [c_int] * 7
        L.gvae_group_norm_ws_bytes.restype = c_int64
        L.gvae_group_norm_fwd.argtypes = [c_void_p, c_int, c_int64, c_int64, c_void_p, c_int, c_int, c_int, c_int,
                                          c_void_p, c_void_p, c_float, c_int] + [c_void_p] * 9
        L.gvae_group_norm_bwd.argtypes = ([c_void_p, c_int, c_int64, c_int64, c_void_p, c_int64, c_int64]
                                          + [c_void_p] * 3 + [c_int] * 4 + [c_void_p] * 4 + [c_int]
                                          + [c_void_p] * 5)
        L.gvae_linear_wgrad8_ws_bytes.argtypes = [c_int64, c_int, c_int]
        L.gvae_linear_wgrad8_ws_bytes.restype = c_int64
        L.gvae_linear_wgrad8.argtypes = [c_void_p, c_int, c_int64, c_void_p, c_void_p, c_int64, c_int, c_int,
                                         c_void_p, c_void_p, c_void_p, c_void_p]
        _bound = L
    return _bound


_device_index = torch._C._cuda_getDevice      # of the current device
_raw_stream = torch._C._cuda_getCurrentRawStream
_empty = torch.empty


def _empty_as(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of t's shape, type and device (empty_like is half a microsecond less than empty)."""
    return torch.empty_like(t) if t.is_contiguous() else _empty(t.shape, dtype=t.dtype, device=t.device)


_any_requires_grad = torch._C._any_requires_grad


def _refuse_recorded(what: str) -> None:
    """Refuses inputs that require grad, whose gradient would be dropped, unless grad mode is off."""
    if torch.is_grad_enabled():
        raise _hip.GvaeHipError(f"{what}: an input requires grad, and the operators here are not recorded by "
                                "autograd: call it under torch.no_grad() or from a torch.autograd.Function")


def _act_code(act: str) -> int:
    code = _ACT.get(act)
    if code is None:
        raise ValueError(f"act must be one of {sorted(_ACT)}, got {act!r}")
    return code


def _on_device(t: torch.Tensor, what: str) -> int:
    """Checks that t is on the current device; returns its index."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise _hip.GvaeHipError(f"{what}: expected a device tensor (the HIP path has no CPU fallback)")
    index = _device_index()
    if t.get_device() != index:
        raise _hip.GvaeHipError(f"{what} on {t.device} but the current device is cuda:{index}: wrap the call in "
                                "torch.cuda.device(...)")
    return index


def _activation(t: torch.Tensor, what: str) -> int:
    """Checks the type and the channels of an activation or gradient; returns its type code."""
    code = _DTYPE.get(t.dtype)
    if code is None:
        raise _hip.GvaeHipError(f"{what}: expected float32, bfloat16 or float16, got {t.dtype}")
    if t.dim() < 1 or t.numel() == 0:
        raise _hip.GvaeHipError(f"{what}: no element in shape {tuple(t.shape)}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise _hip.GvaeHipError(f"{what}: channels must be last and contiguous, got strides {t.stride()}")
    return code


def _small(t, shape: tuple, dtype: torch.dtype, index: int, what: str, name: str):
    """Address of a contiguous side input (None for None) of the given shape and type."""
    if t is None:
        return None
    if t.dtype is not dtype or t.get_device() != index or t.shape != shape or not t.is_contiguous():
        raise _hip.GvaeHipError(f"{what}: {name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on "
                                f"cuda:{index}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _rows_of(t: torch.Tensor, what: str) -> tuple[int, int]:
    """(rows, elements between rows) of an activation seen as a matrix."""
    C = t.shape[-1]
    if t.is_contiguous():
        return t.numel() // C, C
    if t.dim() == 2 and (t.shape[0] == 1 or t.stride(0) >= C):
        return t.shape[0], max(t.stride(0), C)
    raise _hip.GvaeHipError(f"{what}: expected a contiguous tensor or a matrix of evenly spaced rows, got shape "
                            f"{tuple(t.shape)} with strides {t.stride()}")


def _graph_strides(t: torch.Tensor) -> tuple[int, int]:
    """(batch stride, row stride) of (graphs, rows, channels); an axis of length 1 has none of its own."""
    B, N, C = t.shape
    return (t.stride(0) if B > 1 else 0), (t.stride(1) if N > 1 else C)


def _sizes(what: str, *sizes: int) -> None:
    """Refuses sizes that the C entry points' 32-bit arguments cannot hold."""
    if max(sizes) > 0x7fffffff:
        raise _hip.GvaeHipError(f"{what}: sizes {sizes} pass 2^31 - 1")


_NONE = (None, None)


class Checkpoint8:
    """An activation kept in 8 bits: `codes` (..., 16*ceil(C/16)) int8 and `scales` (..., ceil(C/32))
    uint8, value = code * 2^(scale - 127) with one scale per 32 consecutive channels of a row (each
    value off by at most 1/127 of its block's largest; in a block whose largest is under 2^-119 by at most
    2^-127, in one within 1 % of the largest float by at most 1/63).  `channels` is C; `dtype` what
    `read` returns.

    Checkpoint8(codes, scales, channels, dtype) wraps existing tensors, which it keeps."""

    __slots__ = ("_codes", "_scales", "_buf", "_at", "shape", "dtype", "device")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, channels: int,
                 dtype: torch.dtype = torch.bfloat16) -> None:
        C = int(channels)
        lead = tuple(codes.shape[:-1])
        if (C < 1 or codes.dtype != torch.int8 or scales.dtype != torch.uint8
                or tuple(codes.shape) != lead + ((C + 15) // 16 * 16,)
                or tuple(scales.shape) != lead + ((C + 31) // 32,)):
            raise _hip.GvaeHipError(f"Checkpoint8 of {C} channels: codes {tuple(codes.shape)} {codes.dtype}, scales "
                                    f"{tuple(scales.shape)} {scales.dtype}")
        if not (codes.is_contiguous() and scales.is_contiguous()) or codes.device != scales.device:
            raise _hip.GvaeHipError("Checkpoint8: codes and scales must be contiguous and on one device")
        if dtype not in _DTYPE:
            raise _hip.GvaeHipError(f"Checkpoint8: cannot be read as {dtype}")
        if codes.data_ptr() % 16:
            raise _hip.GvaeHipError("Checkpoint8: codes must be 16-byte aligned")
        self._codes, self._scales, self._buf = codes, scales, None
        self._at = (codes.data_ptr(), scales.data_ptr())
        self.shape, self.dtype, self.device = torch.Size(lead + (C,)), dtype, codes.device

    @classmethod
    def _new(cls, shape, rows: int, C: int, device, dtype: torch.dtype) -> "Checkpoint8":
        """Room for a checkpoint: one allocation, the codes first."""
        self = object.__new__(cls)
        n_codes = rows * ((C + 15) // 16 * 16)
        self._buf = buf = _empty(n_codes + rows * ((C + 31) // 32), dtype=torch.uint8, device=device)
        base = buf.data_ptr()
        self._codes = self._scales = None
        self._at = (base, base + n_codes)
        self.shape, self.dtype, self.device = shape, dtype, device
        return self

    def __reduce__(self):
        # (copies and pickles hold their own memory)
        return Checkpoint8, (self.codes, self.scales, self.channels, self.dtype)

    @property
    def channels(self) -> int:
        return self.shape[-1]

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            self._codes = self._buf[:self._at[1] - self._at[0]].view(torch.int8).view(
                self.shape[:-1] + ((self.shape[-1] + 15) // 16 * 16,))
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            self._scales = self._buf[self._at[1] - self._at[0]:].view(
                self.shape[:-1] + ((self.shape[-1] + 31) // 32,))
        return self._scales

    def _check(self, what: str) -> int:
        index = _on_device(self._buf if self._codes is None else self._codes, what)
        if 0 in self.shape:
            raise _hip.GvaeHipError(f"{what}: no element in shape {tuple(self.shape)}")
        return index

    def read(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        """The values the checkpoint stands for, as `dtype` (default: the type that was written);
        exact in bfloat16 and float32."""
        dtype = self.dtype if dtype is None else dtype
        code = _DTYPE.get(dtype)
        if code is None:
            raise _hip.GvaeHipError(f"Checkpoint8.read: cannot be read as {dtype}")
        index = self._check("Checkpoint8.read")
        C = self.shape[-1]
        _sizes("Checkpoint8.read", C)
        out = _empty(self.shape, dtype=dtype, device=self.device)
        rc = (_bound or _bind()).gvae_ckpt8_read(self._at[0], self._at[1], out.numel() // C, C, out.data_ptr(), code, C,
                                                 _raw_stream(index))
        if rc:
            _hip._check(rc)
        return out


def checkpoint8(x: torch.Tensor) -> Checkpoint8:
    """8-bit checkpoint of x (..., C) float32 / bfloat16 / float16: contiguous, or a matrix with any
    row stride of at least C.  A block of 32 channels that holds an infinity or a NaN reads back as NaN."""
    if _any_requires_grad(x):
        _refuse_recorded("checkpoint8")
    index = _on_device(x, "checkpoint8")
    code = _activation(x, "checkpoint8")
    rows, ld = _rows_of(x, "checkpoint8")
    C = x.shape[-1]
    _sizes("checkpoint8", C)
    c = Checkpoint8._new(x.shape, rows, C, x.device, x.dtype)
    rc = (_bound or _bind()).gvae_ckpt8_write(x.data_ptr(), code, rows, C, ld, c._at[0], c._at[1], _raw_stream(index))
    if rc:
        _hip._check(rc)
    return c


class GroupNormOut(NamedTuple):
    y: torch.Tensor             # (graphs, rows, channels), x's type
    mean: torch.Tensor          # (graphs, groups) float32
    rstd: torch.Tensor          # (graphs, groups) float32
    x8: Checkpoint8 | None      # checkpoint of x, if asked for
    y8: Checkpoint8 | None      # checkpoint of y, if asked for


def _norm_sizes(x_shape, groups: int, what: str):
    if len(x_shape) != 3:
        raise _hip.GvaeHipError(f"{what}: expected (graphs, rows, channels), got shape {tuple(x_shape)}")
    B, N, C = x_shape
    _sizes(what, B, N, C, groups)
    if groups < 1 or C % groups:
        raise ValueError(f"{what}: {C} channels do not divide into {groups} groups")
    return B, N, C


def group_norm_act(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, groups: int, *,
                   act: str = "relu", eps: float = 1e-5, rows: torch.Tensor | None = None, keep_x: bool = False,
                   keep_y: bool = False) -> GroupNormOut:
    """act(group_norm(x) * weight + bias) over each graph's live rows and `groups` runs of consecutive
    channels.

    x: (graphs, rows, channels) float32 / bfloat16 / float16, channels contiguous, any row and batch
    strides (expanded axes included).  weight, bias: (channels,) float32 or None.  act: none | relu |
    silu | gelu (the erf form).  rows: live rows per graph (int32), None = all; rows behind them are not read
    and come out 0, a graph without any has mean 0 and variance 0.  keep_x / keep_y: also return 8-bit
    checkpoints of x (dead rows as 0) and of y, the same as `checkpoint8` of them."""
    what = "group_norm_act"
    if _any_requires_grad(x, weight, bias):
        _refuse_recorded(what)
    B, N, C = _norm_sizes(x.shape, groups, what)
    act_code = _act_code(act)
    index = _on_device(x, what)
    code = _activation(x, what)
    batch, row = _graph_strides(x)
    w, b = (_small(weight, (C,), torch.float32, index, what, "weight"),
            _small(bias, (C,), torch.float32, index, what, "bias"))
    live = _small(rows, (B,), torch.int32, index, what, "rows")
    if not eps > 0.0:
        raise ValueError(f"{what}: eps must be positive, got {eps}")
    L, dev = _bound or _bind(), x.device
    y = _empty_as(x)
    mean, rstd = _empty((2, B, groups), dtype=torch.float32, device=dev).unbind(0)
    x8 = Checkpoint8._new(x.shape, B * N, C, dev, x.dtype) if keep_x else None
    y8 = Checkpoint8._new(x.shape, B * N, C, dev, x.dtype) if keep_y else None
    need = L.gvae_group_norm_ws_bytes(0, code, B, N, C, groups, keep_x or keep_y)
    ws = _empty(need, dtype=torch.uint8, device=dev) if need else None
    xc, xs = x8._at if keep_x else _NONE
    yc, ys = y8._at if keep_y else _NONE
    rc = L.gvae_group_norm_fwd(x.data_ptr(), code, batch, row, live, B, N, C, groups, w, b, eps, act_code, y.data_ptr(),
                               mean.data_ptr(), rstd.data_ptr(), xc, xs, yc, ys, ws.data_ptr() if need else None,
                               _raw_stream(index))
    if rc:
        _hip._check(rc)
    return GroupNormOut(y, mean, rstd, x8, y8)


def group_norm_act_backward(dy: torch.Tensor, x, weight: torch.Tensor | None, bias: torch.Tensor | None,
                            mean: torch.Tensor, rstd: torch.Tensor, groups: int, *, act: str = "relu",
                            rows: torch.Tensor | None = None):
    """Gradients of `group_norm_act`: (dx, dweight, dbias), dx of dy's type, the others float32 (summed
    over graphs and rows in a fixed order).  x: the forward's input, of dy's type, or its Checkpoint8;
    mean, rstd: as the forward returned them; weight, bias, groups, act, rows: as given to it.  dy: like x
    of any row and batch strides (a gradient expanded over graphs or rows is read in place; one expanded over
    channels is refused).  dx of dead rows is 0."""
    what = "group_norm_act_backward"
    kept = isinstance(x, Checkpoint8)
    if _any_requires_grad(dy, x, weight, bias):
        _refuse_recorded(what)
    B, N, C = _norm_sizes(dy.shape, groups, what)
    act_code = _act_code(act)
    index = _on_device(dy, what)
    code = _activation(dy, what)
    if x.shape != dy.shape:
        raise _hip.GvaeHipError(f"{what}: input of shape {tuple(x.shape)}, gradient {tuple(dy.shape)}")
    if kept:
        x._check(what)
        xs, xb, xr = None, 0, C
        x8, x8s = x._at
    else:
        _on_device(x, what)
        if x.dtype is not dy.dtype:
            raise _hip.GvaeHipError(f"{what}: input is {x.dtype}, gradient {dy.dtype}")
        _activation(x, what)
        xb, xr = _graph_strides(x)
        xs, x8, x8s = x.data_ptr(), None, None
    db_, dr_ = _graph_strides(dy)
    w, b = (_small(weight, (C,), torch.float32, index, what, "weight"),
            _small(bias, (C,), torch.float32, index, what, "bias"))
    live = _small(rows, (B,), torch.int32, index, what, "rows")
    if mean is None or rstd is None:
        raise _hip.GvaeHipError(f"{what}: needs the mean and rstd of the forward")
    mu, rs = (_small(mean, (B, groups), torch.float32, index, what, "mean"),
              _small(rstd, (B, groups), torch.float32, index, what, "rstd"))
    L, dev = _bound or _bind(), dy.device
    dx = _empty_as(dy)
    dweight, dbias = _empty((2, C), dtype=torch.float32, device=dev).unbind(0)
    ws = _empty(L.gvae_group_norm_ws_bytes(1, code, B, N, C, groups, kept), dtype=torch.uint8, device=dev)
    rc = L.gvae_group_norm_bwd(dy.data_ptr(), code, db_, dr_, xs, xb, xr, x8, x8s, live, B, N, C, groups, w, b, mu, rs,
                               act_code, dx.data_ptr(), dweight.data_ptr(), dbias.data_ptr(), ws.data_ptr(),
                               _raw_stream(index))
    if rc:
        _hip._check(rc)
    return dx, dweight, dbias


def linear_wgrad8(dy: torch.Tensor, x8: Checkpoint8) -> tuple[torch.Tensor, torch.Tensor]:
    """(dweight (O, I), dbias (O)) of a linear layer y = x W^T + b, in dy's type, from its output's
    gradient dy (..., O) and the checkpoint of its input (..., I).  dy: contiguous, or a matrix with any
    row stride of at least O.  Every product is exact (of float32 gradients under 2^-110 what lies below 2^-133
    is dropped), sums are float32 in a fixed order, rounded once."""
    what = "linear_wgrad8"
    if _any_requires_grad(dy):
        _refuse_recorded(what)
    if not isinstance(x8, Checkpoint8):
        raise _hip.GvaeHipError(f"{what}: the input must be a Checkpoint8")
    x8._check(what)
    index = _on_device(dy, what)
    code = _activation(dy, what)
    if dy.dim() < 2 or dy.shape[:-1] != x8.shape[:-1]:
        raise _hip.GvaeHipError(f"{what}: gradient {tuple(dy.shape)} and checkpoint {tuple(x8.shape)} differ in their "
                                "rows")
    rows, ld = _rows_of(dy, what)
    O, I = dy.shape[-1], x8.shape[-1]
    _sizes(what, O, I)
    L, dev = _bound or _bind(), dy.device
    dw = _empty((O, I), dtype=dy.dtype, device=dev)
    db = _empty((O,), dtype=dy.dtype, device=dev)
    ws = _empty(L.gvae_linear_wgrad8_ws_bytes(rows, O, I), dtype=torch.uint8, device=dev)
    rc = L.gvae_linear_wgrad8(dy.data_ptr(), code, ld, x8._at[0], x8._at[1], rows, O, I, dw.data_ptr(), db.data_ptr(),
                              ws.data_ptr(), _raw_stream(index))
    if rc:
        _hip._check(rc)
    return dw, db
