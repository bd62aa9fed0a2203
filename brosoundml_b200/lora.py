"""Python mirror of the reference's ``DecoderLora`` (include/brosoundml/decoder_lora.h:36-164)
over the C ABI: per-AdaIN LoRA adapters on the frozen style -> (gamma, beta)
projections, the shared conditioning gate g(v) = W2 tanh(W1 v), Adam with one
shared step, and the ELRA1 checkpoint. Batched: every clip has its own style and
condition. Every computation runs in libbsml_b200.so.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .decoder import Decoder, _f32, _ptr, _stream

IN_DIM, HIDDEN = 3, 16   # ConditioningGate::in_dim, the gate hidden width (decoder_lora.cpp:141)


class DecoderLora:
    """``DecoderLora::make`` over ``decoder`` (a :class:`Decoder`); the decoder must
    outlive this object."""

    def __init__(self, decoder: Decoder, rank: int = 8, scale: float = 1.0, seed: int = 0):
        L = _lib.lib()
        h = ctypes.c_void_p()
        _lib.check(L.bsml_lora_create(decoder._h, int(rank), float(scale), int(seed), ctypes.byref(h)))
        self._h = h
        self.decoder = decoder
        n, na, r, sd = ctypes.c_int64(), ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
        o1, o2 = ctypes.c_int64(), ctypes.c_int64()
        _lib.check(L.bsml_lora_layout(h, ctypes.byref(n), ctypes.byref(na), ctypes.byref(r), ctypes.byref(sd),
                                      ctypes.byref(o1), ctypes.byref(o2), None, None, None))
        offA = (ctypes.c_int64 * na.value)()
        offB = (ctypes.c_int64 * na.value)()
        C = (ctypes.c_int * na.value)()
        _lib.check(L.bsml_lora_layout(h, None, None, None, None, None, None, ctypes.cast(offA, ctypes.c_void_p),
                                      ctypes.cast(offB, ctypes.c_void_p), ctypes.cast(C, ctypes.c_void_p)))
        self.n_params, self.n_adapters, self.rank, self.style_dim = n.value, na.value, r.value, sd.value
        self.off_W1, self.off_W2 = o1.value, o2.value
        self.off_A, self.off_B, self.adapter_C = list(offA), list(offB), list(C)
        pp, gp = ctypes.c_void_p(), ctypes.c_void_p()
        _lib.check(L.bsml_lora_buffers(h, ctypes.byref(pp), ctypes.byref(gp)))
        self._pp, self._gp = pp.value, gp.value

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is not None and _lib._lib is not None:
            _lib.lib().bsml_lora_destroy(h)
            self._h = None

    # ── the flat parameter / gradient vectors, as torch views of the object's device memory
    def params(self) -> torch.Tensor:
        """View (no copy) of the flat parameter vector: gate W1 [16][3], gate W2 [rank][16],
        then per adapter A [rank][style_dim] (at off_A[a]) and B [2C][rank] (at off_B[a])."""
        return _device_view(self._pp, self.n_params, self.decoder.device)

    def grads(self) -> torch.Tensor:
        """View (no copy) of the flat gradient vector (same layout as :meth:`params`)."""
        return _device_view(self._gp, self.n_params, self.decoder.device)

    @property
    def scale(self) -> float:
        s, st = ctypes.c_float(), ctypes.c_int()
        _lib.check(_lib.lib().bsml_lora_state(self._h, ctypes.byref(s), ctypes.byref(st)))
        return s.value

    @property
    def step(self) -> int:
        s, st = ctypes.c_float(), ctypes.c_int()
        _lib.check(_lib.lib().bsml_lora_state(self._h, ctypes.byref(s), ctypes.byref(st)))
        return st.value

    # ── DecoderLora::forward / backward / zero_grad / adam_step / save / load
    def forward(self, params, asr, F0, N, ref_s, cond, har=None, audio=None):
        params, asr, F0, N, ref_s, cond, har = map(_f32, (params, asr, F0, N, ref_s, cond, har))
        B, _, T = asr.shape
        frames = 0 if har is None else har.shape[2]
        if audio is None:
            audio = torch.empty((B, self.decoder.audio_len(T, frames if har is not None else None)),
                                device=self.decoder.device)
        self._borrowed = params   # the engine reads the weights again in the backward
        _lib.check(_lib.lib().bsml_lora_forward(self._h, B, T, _ptr(params), _ptr(asr), _ptr(F0), _ptr(N),
                                                _ptr(ref_s), ref_s.shape[-1], _ptr(har), frames, _ptr(cond),
                                                _ptr(audio), _stream()))
        return audio

    def backward(self, daudio) -> None:
        _lib.check(_lib.lib().bsml_lora_backward(self._h, _ptr(_f32(daudio)), _stream()))

    def zero_grad(self) -> None:
        _lib.check(_lib.lib().bsml_lora_zero_grad(self._h, _stream()))

    def adam_step(self, lr: float, beta1: float = 0.9, beta2: float = 0.999, eps: float = 1e-8) -> None:
        _lib.check(_lib.lib().bsml_lora_adam_step(self._h, lr, beta1, beta2, eps, _stream()))

    def save(self, path: str, full_state: bool = False) -> None:
        """ELRA1 checkpoint; full_state adds Adam's moments and step after it (the
        file stays readable by the plain-format readers)."""
        fn = _lib.lib().bsml_lora_save_state if full_state else _lib.lib().bsml_lora_save
        _lib.check(fn(self._h, str(path).encode()))

    def load(self, path: str, full_state: bool = False) -> None:
        fn = _lib.lib().bsml_lora_load_state if full_state else _lib.lib().bsml_lora_load
        _lib.check(fn(self._h, str(path).encode()))


class _DeviceBuffer:
    def __init__(self, ptr: int, n: int):
        self.__cuda_array_interface__ = {"shape": (n,), "typestr": "<f4", "data": (ptr, False), "version": 3}


def _device_view(ptr: int, n: int, device) -> torch.Tensor:
    return torch.as_tensor(_DeviceBuffer(ptr, n), device=device)


class ConvLora:
    """Conv-weight LoRA (the fine-tune of every conv weight; no counterpart in the reference): a rank-r
    adapter W + scale * B A on every Conv1d / ConvTranspose1d weight of ``decoder``,
    base weights frozen. A weight stored (d0, d1, k) is viewed as [d0][d1*k];
    A [rank][d1*k] starts N(0, 0.01), B [d0][rank] starts at zero."""

    def __init__(self, decoder: Decoder, rank: int = 8, scale: float = 2.0, seed: int = 0):
        L = _lib.lib()
        h = ctypes.c_void_p()
        _lib.check(L.bsml_convlora_create(decoder._h, int(rank), float(scale), int(seed), ctypes.byref(h)))
        self._h, self.decoder, self.rank, self.scale = h, decoder, int(rank), float(scale)
        n, nw = ctypes.c_int64(), ctypes.c_int()
        _lib.check(L.bsml_convlora_layout(h, ctypes.byref(n), ctypes.byref(nw), None, None, None, None, None))
        arrs = [(ctypes.c_int64 * nw.value)(), (ctypes.c_int * nw.value)(), (ctypes.c_int * nw.value)(),
                (ctypes.c_int64 * nw.value)(), (ctypes.c_int64 * nw.value)()]
        _lib.check(L.bsml_convlora_layout(h, None, None, *[ctypes.cast(a, ctypes.c_void_p) for a in arrs]))
        self.n_params = n.value
        self.weights = [dict(w=w, rows=r, cols=c, offA=a, offB=b) for w, r, c, a, b in zip(*[list(a) for a in arrs])]
        pp, gp = ctypes.c_void_p(), ctypes.c_void_p()
        _lib.check(L.bsml_convlora_buffers(h, ctypes.byref(pp), ctypes.byref(gp)))
        self._pp, self._gp = pp.value, gp.value

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is not None and _lib._lib is not None:
            _lib.lib().bsml_convlora_destroy(h)
            self._h = None

    def params(self) -> torch.Tensor:
        return _device_view(self._pp, self.n_params, self.decoder.device)

    def grads(self) -> torch.Tensor:
        return _device_view(self._gp, self.n_params, self.decoder.device)

    def forward(self, params, asr, F0, N, style, har=None, audio=None):
        params, asr, F0, N, style, har = map(_f32, (params, asr, F0, N, style, har))
        B, _, T = asr.shape
        frames = 0 if har is None else har.shape[2]
        if audio is None:
            audio = torch.empty((B, self.decoder.audio_len(T, frames if har is not None else None)),
                                device=self.decoder.device)
        _lib.check(_lib.lib().bsml_convlora_forward(self._h, B, T, _ptr(params), _ptr(asr), _ptr(F0), _ptr(N),
                                                    _ptr(style), _ptr(har), frames, _ptr(audio), _stream()))
        return audio

    def backward(self, daudio) -> None:
        _lib.check(_lib.lib().bsml_convlora_backward(self._h, _ptr(_f32(daudio)), _stream()))

    def zero_grad(self) -> None:
        _lib.check(_lib.lib().bsml_convlora_zero_grad(self._h, _stream()))

    def adam_step(self, lr: float, beta1: float = 0.9, beta2: float = 0.999, eps: float = 1e-8) -> None:
        _lib.check(_lib.lib().bsml_convlora_adam_step(self._h, lr, beta1, beta2, eps, _stream()))

    def save(self, path: str) -> None:
        """Full training state (ECLR1): A, B, Adam moments and step."""
        _lib.check(_lib.lib().bsml_convlora_save(self._h, str(path).encode()))

    def load(self, path: str) -> None:
        _lib.check(_lib.lib().bsml_convlora_load(self._h, str(path).encode()))


# ── the projection of many requests, and dropout (any of float32, bfloat16, float16)
DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _refuse(name: str, t, shape, dtype, device, strided: bool):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"brosoundml: {name}: expected a CUDA tensor")
    if t.dtype is not dtype:
        raise TypeError(f"brosoundml: {name}: expected {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"brosoundml: {name}: on {t.device}, expected {device}")
    if t.shape != shape:
        raise ValueError(f"brosoundml: {name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    raise ValueError(f"brosoundml: {name}: expected {'contiguous rows' if strided else 'a contiguous tensor'}, "
                     f"got strides {tuple(t.stride())}")


def _whole(name: str, t, shape, dtype, device) -> int:
    """The address of ``t``, a contiguous CUDA tensor of this shape, type and device."""
    try:
        if t.dtype is dtype and t.is_contiguous() and t.shape == shape and t.device == device:
            return t.data_ptr()
    except AttributeError:
        pass
    _refuse(name, t, shape, dtype, device, False)


def _rows(name: str, t, shape, dtype, device):
    """The address and row stride of ``t``, whose rows are contiguous, at any stride that does not
    overlap them (of a single row, whose stride means nothing: its length)."""
    try:
        if t.dtype is dtype and t.shape == shape and t.device == device:
            if t.is_contiguous() or shape[0] <= 1 and (shape[1] <= 1 or t.stride(1) == 1):
                return t.data_ptr(), shape[1] or 1
            if (shape[1] <= 1 or t.stride(1) == 1) and t.stride(0) >= shape[1]:
                return t.data_ptr(), t.stride(0)
    except AttributeError:
        pass
    _refuse(name, t, shape, dtype, device, True)


def _matrix(name: str, t):
    """``t``'s shape, type and device, for the operands that follow."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dim() != 2 or t.dtype not in DTYPE:
        raise TypeError(f"brosoundml: {name}: expected a 2-D CUDA tensor of float32, bfloat16 or float16")
    return t.shape, t.dtype, t.device


def _rng(rng, p, device):
    return None if rng is None and p == 0 else _whole("rng", rng, (2,), torch.int64, device)


def _call(name, device, *args):
    """The entry point ``name(*args, stream)`` on ``device`` and its current stream."""
    fn, index = getattr(_lib.lib(), name), device.index
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc)


def _adapter_args(W, A, B, row_ids, scale, dropout, rng, zero_padding, rows, dtype, device):
    """Checks what the forward and the backward share: the shape and the addresses."""
    try:
        (cout, cin), (n, rank, _) = W.shape, A.shape
    except (AttributeError, ValueError):
        raise TypeError("brosoundml: expected tensors W (cout, cin), A (adapters, rank, cin), "
                        "B (adapters, cout, rank)") from None
    return (_lib.BsmlMultiLoraShape(DTYPE[dtype], rows, cin, cout, rank, n, zero_padding, dropout), cin, cout, rank,
            _whole("W", W, (cout, cin), dtype, device), _whole("A", A, (n, rank, cin), dtype, device),
            _whole("B", B, (n, cout, rank), dtype, device), _whole("row_ids", row_ids, (rows,), torch.int32, device),
            None if scale is None else _whole("scale", scale, (n,), torch.float32, device), _rng(rng, dropout, device))


def multi_lora_forward(x, W, A, B, row_ids, bias=None, scale=None, dropout: float = 0.0, rng=None, y=None, h=None):
    """The shared projection with each row's own adapter (``bsml_multilora_forward``):
    ``y[m] = W x[m] + bias + B[a] h[m]``, ``h[m] = scale[a] / (1 - p) A[a] (keep * x[m])``, a = row_ids[m].

    x (rows, cin), W (cout, cin), bias (cout), A (adapters, rank, cin), B (adapters, cout, rank) of one
    type; row_ids (rows,) int32: an adapter, -1 the shared projection alone, below -1 a padding row; scale
    (adapters,) float32, 1 by default. x and y may be rows of a wider tensor. ``y``: given, its padding
    rows are left as they were; else a new tensor, in which they are zero. ``dropout`` > 0 drops the
    adapters' input, with ``rng`` = int64 {seed, offset} on the device. ``h`` (rows, rank) float32, when
    given, receives what :func:`multi_lora_backward` needs. Works on ``x``'s device and its current stream,
    with scratch of its own that later calls use again (:func:`release_scratch`). A kernel whose bounded wait runs
    out leaves its outputs incomplete and a code that ``bsml_device_error`` reads."""
    (rows, _), dtype, device = _matrix("x", x)
    shape, cin, cout, rank, W, A, B, ids, scale, rng = _adapter_args(W, A, B, row_ids, scale, dropout, rng, y is None,
                                                                     rows, dtype, device)
    at_x, ldx = _rows("x", x, (rows, cin), dtype, device)
    if bias is not None:
        bias = _whole("bias", bias, (cout,), dtype, device)
    if h is not None:
        h = _whole("h", h, (rows, rank), torch.float32, device)
    if y is None:
        y = x.new_empty((rows, cout))
        at_y, ldy = y.data_ptr(), cout
    else:
        at_y, ldy = _rows("y", y, (rows, cout), dtype, device)
    _call("bsml_multilora_forward", device, shape, at_x, ldx, W, bias, A, B, scale, ids, rng, at_y, ldy, h)
    return y


def multi_lora_backward(dy, x, W, A, B, row_ids, h, scale=None, dropout: float = 0.0, rng=None, dx=None, dA=None,
                        dB=None, want_dx: bool = True, want_adapters: bool = True):
    """Gradients of :func:`multi_lora_forward` (``bsml_multilora_backward``) from dy (rows, cout), with the
    forward's arguments and its ``h``: a dict of dx (rows, cin), dA and dB (the layouts and type of A and B,
    overwritten; zero for an adapter without rows). W is frozen. dx, dA, dB may be given as preallocated
    outputs; a given dx keeps its padding rows, a new one has zeros there. x is read for dA alone and ``h``
    for dB alone: either may be None where that is not wanted."""
    (rows, _), dtype, device = _matrix("dy", dy)
    shape, cin, cout, rank, at_W, at_A, at_B, ids, scale, rng = _adapter_args(
        W, A, B, row_ids, scale, dropout, rng, dx is None, rows, dtype, device)
    at_dy, lddy = _rows("dy", dy, (rows, cout), dtype, device)
    at_x = at_h = at_dx = at_dA = at_dB = None
    ldx = lddx = 0
    if dx is not None:
        at_dx, lddx = _rows("dx", dx, (rows, cin), dtype, device)
    elif want_dx:
        dx = dy.new_empty((rows, cin))
        at_dx, lddx = dx.data_ptr(), cin
    if dA is not None:
        at_dA = _whole("dA", dA, A.shape, dtype, device)
    elif want_adapters:
        dA = torch.empty_like(A)
        at_dA = dA.data_ptr()
    if dB is not None:
        at_dB = _whole("dB", dB, B.shape, dtype, device)
    elif want_adapters:
        dB = torch.empty_like(B)
        at_dB = dB.data_ptr()
    if x is not None or dA is not None:
        at_x, ldx = _rows("x", x, (rows, cin), dtype, device)
    if h is not None or dB is not None:
        at_h = _whole("h", h, (rows, rank), torch.float32, device)
    _call("bsml_multilora_backward", device, shape, at_dy, lddy, at_x, ldx, at_W, at_A, at_B, scale, ids, rng,
          at_h, at_dx, lddx, at_dA, at_dB)
    return dict(dx=dx, dA=dA, dB=dB)


def release_scratch() -> None:
    """Gives back to the current device the scratch that no call of :func:`multi_lora_forward` or
    :func:`multi_lora_backward` uses any more (``bsml_multilora_release_scratch``); later calls take it anew."""
    torch.cuda.synchronize()
    _lib.check(_lib.lib().bsml_multilora_release_scratch())


def dropout_forward(x, p: float, rng, residual=None, y=None):
    """``residual + keep / (1 - p) * x`` (``bsml_dropout_forward``) over x (rows, cols), whose rows may lie in a
    wider tensor. ``rng``: int64 {seed, offset} on the device; the mask is a function of it, the row and the
    column alone, in steps of p of 2^-16, and is not stored. ``y`` may be ``x`` or ``residual``."""
    shape, dtype, device = _matrix("x", x)
    at_x, ldx = _rows("x", x, shape, dtype, device)
    at_r, ldr = (None, 0) if residual is None else _rows("residual", residual, shape, dtype, device)
    if y is None:
        y = x.new_empty(shape)
        at_y, ldy = y.data_ptr(), shape[1] or 1
    else:
        at_y, ldy = _rows("y", y, shape, dtype, device)
    _call("bsml_dropout_forward", device, DTYPE[dtype], at_x, ldx, at_r, ldr, shape[0], shape[1], p,
          _rng(rng, p, device), at_y, ldy)
    return y


def dropout_backward(dy, p: float, rng, dx=None):
    """``keep / (1 - p) * dy`` with the mask of :func:`dropout_forward` under the same ``rng``
    (``bsml_dropout_backward``); the residual's gradient is dy itself. ``dx`` may be ``dy``."""
    shape, dtype, device = _matrix("dy", dy)
    at_dy, lddy = _rows("dy", dy, shape, dtype, device)
    if dx is None:
        dx = dy.new_empty(shape)
        at_dx, lddx = dx.data_ptr(), shape[1] or 1
    else:
        at_dx, lddx = _rows("dx", dx, shape, dtype, device)
    _call("bsml_dropout_backward", device, DTYPE[dtype], at_dy, lddy, shape[0], shape[1], p,
          _rng(rng, p, device), at_dx, lddx)
    return dx
