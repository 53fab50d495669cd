"""8-bit activation checkpoints: what a training step keeps of its forward pass for its backward pass, written, read back
and used there (``camal_act_*`` of libcamal_hip.so).

Where torch's autograd keeps the fp32 convolution output and the fp32 activation of every ConvBlock
(camal_resnet.py:81-86 under torch_trainer.py:288-291), a checkpoint keeps the normalised values in one byte each, with
one power-of-two scale byte per 32 channels of a timestep, and serves both uses that the backward pass has for them: the
BatchNorm + ReLU backward (``norm_backward``) and the weight gradient of the layer that reads the activation
(``conv_weight_grad``; one tap = a linear layer).  ``TrainEngine(..., act_checkpoint="int8" | "e4m3")`` runs whole training
steps on them.

Tensors are ``[window, time, channel]`` on one GPU, channels in {32, 64, 128, 256}; the calls are asynchronous on the
current stream of that GPU.  They are the parts of a backward pass written out by hand: none of them is recorded by autograd,
whatever requires a gradient among its arguments, and what they return does not require one.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib

BLOCK = 32  # channels that share a scale
CHANNELS = (32, 64, 128, 256)
FORMATS = {"int8": (torch.int8, _lib.ACT_INT8), "e4m3": (torch.float8_e4m3fn, _lib.ACT_E4M3)}


@dataclass(frozen=True)
class ActivationCheckpoint:
    """``codes`` [B, L, C] (``torch.int8`` or ``torch.float8_e4m3fn``) and ``scales`` [B, L, C / 32] (``torch.uint8``):
    the normalised value of an element is ``code * 2 ** (scale - 127)``, scales from 1 on; 255 goes with codes 0 and makes the
    block's values NaN."""
    codes: torch.Tensor
    scales: torch.Tensor

    def __post_init__(self):
        if self.codes.dtype not in (torch.int8, torch.float8_e4m3fn) or self.scales.dtype != torch.uint8:
            raise ValueError("codes are torch.int8 or torch.float8_e4m3fn, scales torch.uint8")
        if self.codes.dim() != 3 or self.codes.shape[-1] not in CHANNELS:
            raise ValueError(f"codes are [windows, time, channels] with channels in {CHANNELS}, got {tuple(self.codes.shape)}")
        if tuple(self.scales.shape) != (*self.codes.shape[:2], self.codes.shape[2] // BLOCK):
            raise ValueError(f"scales are [windows, time, channels / {BLOCK}], got {tuple(self.scales.shape)}")
        if self.codes.device != self.scales.device:
            raise ValueError("codes and scales are on different devices")

    @property
    def shape(self):
        return self.codes.shape

    @property
    def device(self):
        return self.codes.device

    @property
    def fmt(self):
        return "int8" if self.codes.dtype == torch.int8 else "e4m3"

    @property
    def nbytes(self):
        return self.codes.numel() + self.scales.numel()


def _device(t):
    if not t.is_cuda:
        raise _lib.CamalHipError(f"activation checkpoints live on MI355X only (device={str(t.device)!r}); there is no CPU path.")
    return t.device


def _rows(t):
    """The tensor as the kernels read it: rows behind each other, 16-byte aligned (a copy only if it is not)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _floats(t, shape, device, name):
    if not torch.is_tensor(t) or t.dtype != torch.float32 or t.shape != shape or t.device != device:
        raise ValueError(f"{name}: expected a float32 tensor of shape {tuple(shape)} on {device}")
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else _rows(t)


def _ckpt(c, device, name, shape=None, fmt=None):
    if not isinstance(c, ActivationCheckpoint) or c.device != device or (shape is not None and tuple(c.shape) != tuple(shape)):
        raise ValueError(f"{name}: expected an ActivationCheckpoint{'' if shape is None else f' of shape {tuple(shape)}'} on {device}")
    if fmt is not None and c.fmt != fmt:
        raise ValueError(f"{name}: both branches must have one format")
    return _rows(c.codes), _rows(c.scales)


def _skip(skip, ckpt):
    """(codes, scales, gamma, beta) of the skip branch, or four None."""
    if skip is None:
        return None, None, None, None
    other, gamma, beta = skip
    codes, scales = _ckpt(other, ckpt.device, "skip", ckpt.shape, ckpt.fmt)
    n = (ckpt.shape[-1],)
    return codes, scales, _floats(gamma, n, ckpt.device, "skip gamma"), _floats(beta, n, ckpt.device, "skip beta")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(device, fn, *args):
    """``fn(*args, stream)`` on the tensors' GPU and its current stream."""
    stream = torch._C._cuda_getCurrentRawStream(device.index)
    if torch.cuda.current_device() == device.index:
        code = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            code = fn(*args, stream)
    if code:
        _lib.check(code)


def _new(z, dtype):
    """An unwritten checkpoint of z's shape (which the caller has looked over)."""
    kept = object.__new__(ActivationCheckpoint)
    object.__setattr__(kept, "codes", torch.empty_like(z, dtype=dtype))
    object.__setattr__(kept, "scales", z.new_empty((z.shape[0], z.shape[1], z.shape[2] // BLOCK), dtype=torch.uint8))
    return kept


def write(z, mean, invstd, gamma, beta, relu=True, fmt="int8", skip=None):
    """Normalise ``z`` [B, L, C] with the batch statistics, scale, shift, ReLU, add the skip branch; keep it in 8 bits.

    ``skip``: ``(z, mean, invstd, gamma, beta)`` of a branch that is added without a ReLU (camal_resnet.py:56-58).
    -> ``(out, checkpoint)``, or ``(out, checkpoint, skip_checkpoint)`` with a skip branch; ``out`` is the fp32
    activation, computed from ``z`` and not from the codes."""
    if fmt not in FORMATS:
        raise ValueError(f"fmt must be one of {tuple(FORMATS)}")
    if not torch.is_tensor(z) or z.dim() != 3 or z.shape[-1] not in CHANNELS:
        raise ValueError(f"z is [windows, time, channels] with channels in {CHANNELS}")
    dev, (B, L, ch) = _device(z), z.shape
    dtype, code = FORMATS[fmt]
    n = (ch,)
    a = [_floats(z, z.shape, dev, "z"), _floats(mean, n, dev, "mean"), _floats(invstd, n, dev, "invstd"),
         _floats(gamma, n, dev, "gamma"), _floats(beta, n, dev, "beta")]
    r = [None] * 5
    if skip is not None:
        names = ("skip z", "skip mean", "skip invstd", "skip gamma", "skip beta")
        r = [_floats(t, s, dev, name) for t, s, name in zip(skip, (z.shape, n, n, n, n), names, strict=True)]
    out, kept = torch.empty_like(a[0]), _new(a[0], dtype)
    if skip is None:
        _call(dev, _lib.load().camal_act_write, *map(_ptr, a), int(bool(relu)), *r, B * L, ch, code, out.data_ptr(),
              kept.codes.data_ptr(), kept.scales.data_ptr(), None, None)
        return out, kept
    side = _new(a[0], dtype)
    _call(dev, _lib.load().camal_act_write, *map(_ptr, a), int(bool(relu)), *map(_ptr, r), B * L, ch, code, out.data_ptr(),
          kept.codes.data_ptr(), kept.scales.data_ptr(), side.codes.data_ptr(), side.scales.data_ptr())
    return out, kept, side


def read(ckpt, gamma=None, beta=None, relu=True, skip=None):
    """The values that a checkpoint stands for, fp32 [B, L, C]: the normalised values (no ``gamma``), or the activation
    ``[relu](gamma x + beta)`` plus that of ``skip = (checkpoint, gamma, beta)``."""
    codes, scales = _ckpt(ckpt, _device(ckpt.codes), "checkpoint")
    dev, (B, L, ch) = ckpt.device, ckpt.shape
    if gamma is None and (beta is not None or skip is not None):
        raise ValueError("beta and skip need gamma")
    g = b = None
    if gamma is not None:
        g, b = _floats(gamma, (ch,), dev, "gamma"), _floats(beta, (ch,), dev, "beta")
    r = _skip(skip, ckpt)
    out = torch.empty((B, L, ch), dtype=torch.float32, device=dev)
    _call(dev, _lib.load().camal_act_read, codes.data_ptr(), scales.data_ptr(), FORMATS[ckpt.fmt][1], B * L, ch, _ptr(g), _ptr(b),
          int(bool(relu) and g is not None), *map(_ptr, r), out.data_ptr())
    return out


def norm_backward(da, ckpt, invstd, gamma, beta, relu=True):
    """Backward of BatchNorm (+ ReLU) from the checkpoint of its normalised values -> ``(dz, dgamma, dbeta)``.

    ``da``: gradient of the output, [B, L, C]; or [B, C], the gradient of each window's mean over time (camal_resnet.py:23),
    which every timestep shares.  ``invstd``, ``gamma``, ``beta``: those that the checkpoint was written with."""
    codes, scales = _ckpt(ckpt, _device(ckpt.codes), "checkpoint")
    dev, (B, L, ch) = ckpt.device, ckpt.shape
    pooled = torch.is_tensor(da) and da.dim() == 2
    da = _floats(da, (B, ch) if pooled else (B, L, ch), dev, "da")
    p = [_floats(t, (ch,), dev, n) for t, n in ((invstd, "invstd"), (gamma, "gamma"), (beta, "beta"))]
    lib = _lib.load()
    dz, dgamma, dbeta = torch.empty((B, L, ch), dtype=torch.float32, device=dev), torch.empty_like(p[1]), torch.empty_like(p[1])
    ws = torch.empty(lib.camal_act_norm_bwd_workspace_bytes(B * L, ch), dtype=torch.uint8, device=dev)
    _call(dev, lib.camal_act_norm_bwd, da.data_ptr(), int(pooled), codes.data_ptr(), scales.data_ptr(), FORMATS[ckpt.fmt][1], B, L, ch,
          *map(_ptr, p), int(bool(relu)), dz.data_ptr(), dgamma.data_ptr(), dbeta.data_ptr(), ws.data_ptr(), ws.numel())
    return dz, dgamma, dbeta


def conv_weight_grad(dz, ckpt, kernel_size, gamma, beta, relu=True, skip=None, zero_pad=False):
    """Weight gradient [Cout, Cin, kernel_size] of a Conv1d from ``dz`` [B, L, Cout] and the checkpoint of its input.

    The input is ``read(ckpt, gamma, beta, relu, skip)`` rounded to bf16; outside the window the edge samples repeat
    (camal_resnet.py:83), or are zeros with ``zero_pad`` (classifiers/resnet.py:62).  ``kernel_size`` is odd and at most 63; 1
    is a linear layer."""
    codes, scales = _ckpt(ckpt, _device(ckpt.codes), "checkpoint")
    dev, (B, L, cin) = ckpt.device, ckpt.shape
    if not torch.is_tensor(dz) or dz.dim() != 3 or dz.shape[-1] not in CHANNELS:
        raise ValueError(f"dz is [windows, time, channels] with channels in {CHANNELS}")
    cout, ks = dz.shape[-1], int(kernel_size)
    if ks != kernel_size or not 1 <= ks <= 63 or ks % 2 == 0:
        raise _lib.CamalHipError("kernel_size must be odd and in 1..63")
    dz = _floats(dz, (B, L, cout), dev, "dz")
    g, b = _floats(gamma, (cin,), dev, "gamma"), _floats(beta, (cin,), dev, "beta")
    r = _skip(skip, ckpt)
    lib = _lib.load()
    dw = torch.empty((cout, cin, ks), dtype=torch.float32, device=dev)
    ws = torch.empty(lib.camal_act_wgrad_workspace_bytes(B, L, cin, cout, ks), dtype=torch.uint8, device=dev)
    _call(dev, lib.camal_act_wgrad, dz.data_ptr(), codes.data_ptr(), scales.data_ptr(), FORMATS[ckpt.fmt][1], B, L, cin, cout, ks,
          g.data_ptr(), b.data_ptr(), int(bool(relu)), *map(_ptr, r), int(bool(zero_pad)), dw.data_ptr(), ws.data_ptr(), ws.numel())
    return dw
