"""Choice of experts and 8-bit floating point products on CUDA torch tensors.

The device entry points of include/llambda_cuda.h for routers and weights other
than llambda's own two architectures and GGML blocks: `route_experts` turns
router logits into experts and weights, `fp8_quantize` turns activations into
e4m3 with a scale per row and 128 columns, `Fp8ProjectionSession` and
`Fp8MoeSession` multiply them by e4m3 weights with a scale per 128 x 128 block.
As everywhere in this package there is no CPU fallback.  An argument whose type,
shape, strides or device is wrong is a ValueError; what the library refuses
(overlaps, sizes, routing options) and a call that fails are LlambdaCudaErrors.

Device calls run on `stream` (default: the current stream of the tensors'
device); memory they return or need for working is allocated on that stream, so
they may be captured into a CUDA graph and overlap on different streams.  A call
does not wait for other streams: whoever passes a `stream` orders it after what
writes the inputs.  The inputs may be dropped right after the call when `stream`
is a torch.cuda.Stream; with a raw handle or an ExternalStream they are kept until
the stream is done with them.  An `out`
that overlaps an input or a session's weights is refused (columns of one buffer
do not overlap).  Torch
is only plumbing here (allocation and streams).  The inputs are read, never
differentiated: a tensor that requires grad is refused while autograd records,
and one with a tangent in forward mode.
"""
from __future__ import annotations

import ctypes as C
import functools

import numpy as np

from . import _native as N

BLOCK = 128  # columns (and weight rows) per scale


# A one-token call is a few microseconds of GPU time, so what a call does on the
# host is kept short: torch, its types, the library and the lookup of the current
# stream are bound once, by the first call that needs them.
_t = _lib = _raw_stream = _forward = None
_FLOATS = _FP8 = _INT = _F32 = ()


def _torch():
    global _t, _raw_stream, _forward, _FLOATS, _FP8, _INT, _F32
    if _t is None:
        import torch
        import torch.autograd.forward_ad as _forward
        _FLOATS = (torch.float32, torch.bfloat16)
        _FP8 = (torch.float8_e4m3fn, torch.uint8)
        _INT, _F32 = (torch.int32,), (torch.float32,)
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                              lambda index: torch.cuda.current_stream(index).cuda_stream)
        _t = torch
    return _t


def _library():
    global _lib
    if _lib is None:
        _lib = N.lib()
    return _lib


def _check(status: int) -> None:
    if status != 0:
        raise N.LlambdaCudaError(N.last_error() or "the call failed")


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _pad(n: int, m: int) -> int:
    return -(-n // m) * m


def _device_tensor(t, name: str, dtypes, shape, device=None, contiguous=False):
    """Checks a CUDA tensor: type, shape (None: any), unit stride along the last axis."""
    torch = _t or _torch()
    try:  # the usual case in few steps; what fails it is looked at below
        if (t.is_cuda and t.dtype in dtypes and t.shape == shape and t.is_contiguous()
                and t.numel() and (device is None or t.device == device)
                and not t.requires_grad and _forward._current_level < 0):
            return t
    except AttributeError:
        pass
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d)[6:] for d in dtypes)}, "
                         f"got {str(t.dtype)[6:]}")
    got = t.shape
    if len(got) != len(shape) or any(w is not None and w != g for w, g in zip(shape, got)):
        raise ValueError(f"{name} has shape {tuple(got)}, expected "
                         f"{tuple('any' if s is None else s for s in shape)}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires grad; these operators have no backward pass")
    if _forward._current_level >= 0 and _forward.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} has a tangent; these operators have no derivative")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, not {device}")
    if 0 in got:
        raise ValueError(f"{name} is empty (a positive token count is required)")
    if contiguous:
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    elif got[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must have unit stride along its last axis")
    return t


def _matrix(t, name: str, cols=None, device=None):
    """Checks a float32 or bfloat16 operand [tokens][cols]; its (rows, columns, row stride)."""
    if _t is None:
        _torch()
    try:
        rows, width = t.shape
    except (AttributeError, ValueError, TypeError):
        rows = width = None
    if cols is None:
        cols = width
    _device_tensor(t, name, _FLOATS, (rows, cols), device)
    return rows, cols, t.stride(0) if rows > 1 else cols


def _tag(dtype) -> int:
    return N.TYPE_F32 if dtype is _FLOATS[0] else N.TYPE_BF16


def _on(stream, device, operands, allocate):
    """(raw handle of the call's stream, allocate()'s result with that stream
    current, so that what the call allocates belongs to it).  The memory of
    `operands` is not given out again before a `stream` is done with it; a raw
    handle's owner may destroy its stream first, so there the caller keeps them."""
    if stream is None:
        return _raw_stream(device.index), allocate()
    torch = _torch()
    if not hasattr(stream, "cuda_stream"):
        stream = torch.cuda.ExternalStream(int(stream), device=device)
    if stream.device != device:
        raise ValueError(f"the stream is on {stream.device}, not {device}")
    if not isinstance(stream, torch.cuda.ExternalStream):
        for t in operands:
            if t is not None:
                t.record_stream(stream)
    with torch.cuda.stream(stream):
        return stream.cuda_stream, allocate()


def _out(out, rows: int, cols: int, dtype, device, name="out"):
    if out is None:
        if dtype not in _FLOATS:
            raise ValueError(f"{name} must be float32 or bfloat16, got {str(dtype)[6:]}")
        return _t.empty((rows, cols), dtype=dtype, device=device), cols
    _device_tensor(out, name, _FLOATS, (rows, cols), device)
    return out, out.stride(0) if rows > 1 else cols


# ------------------------------------------------------------------ routing


@functools.lru_cache(maxsize=256)  # descriptors are constants, built once per set of options
def _route_desc(experts, top_k, score, groups, top_groups, group_top, renormalise, weight_scale):
    scores = {"softmax": N.SCORE_SOFTMAX, "sigmoid": N.SCORE_SIGMOID}
    if score not in scores:
        raise ValueError(f"score must be 'softmax' or 'sigmoid', got {score!r}")
    if not 1 <= top_k <= experts:
        raise ValueError(f"top_k must be in 1..{experts}, got {top_k}")
    return C.pointer(N.RouteDesc(experts, top_k, scores[score], groups, top_groups, group_top,
                                 int(bool(renormalise)), weight_scale))


def route_experts(logits, top_k: int, *, score: str = "softmax", bias=None, groups: int = 1,
                  top_groups: int = 1, group_top: int = 1, renormalise: bool = True,
                  weight_scale: float = 1.0, stream=None):
    """(selected int32 [T, top_k], weights float32 [T, top_k]) of router logits
    [T, experts] (float32 or bfloat16 CUDA tensor, rows of any stride; or a
    numpy array, then numpy arrays come back).

    Scores are the softmax or sigmoid of a token's logits; the choice goes by
    score + bias (float32 [experts]), within the `top_groups` best of `groups`
    equal groups, a group's rank being its largest choice (group_top 1) or the
    sum of its two largest (2).  Experts come in decreasing order, equal ones by
    index; choices are compared in 64 bits, and by their logits where that does
    not tell them apart.  Weights are the scores without
    bias, divided by their sum with `renormalise`, times `weight_scale`.  An
    expert with a logit of -inf has score 0 and is chosen last."""
    if not hasattr(logits, "data_ptr"):
        return _route_host(logits, bias, _route_desc(
            np.shape(logits)[-1], top_k, score, groups, top_groups, group_top, renormalise,
            weight_scale))
    T, E, ld = _matrix(logits, "logits")
    dev = logits.device
    if bias is not None:
        _device_tensor(bias, "bias", _F32, (E,), dev)
    desc = _route_desc(E, top_k, score, groups, top_groups, group_top, renormalise, weight_scale)
    raw, (selected, weights) = _on(stream, dev, (logits, bias), lambda: (
        _t.empty((T, top_k), dtype=_t.int32, device=dev),
        _t.empty((T, top_k), dtype=_t.float32, device=dev)))
    _check((_lib or _library()).llambda_cuda_route_device(
        desc, _tag(logits.dtype), logits.data_ptr(), ld,
        bias.data_ptr() if bias is not None else None, T, selected.data_ptr(),
        weights.data_ptr(), raw))
    return selected, weights


def _route_host(logits, bias, desc):
    logits = N._f32(logits)
    E, k = desc.contents.experts, desc.contents.top_k
    if logits.ndim != 2 or 0 in logits.shape:
        raise ValueError("logits must be [tokens][experts] with a positive token count")
    if bias is not None:
        bias = N._f32(bias)
        if bias.shape != (E,):
            raise ValueError(f"bias must have shape ({E},)")
    T = logits.shape[0]
    selected, weights = np.empty((T, k), np.int32), np.empty((T, k), np.float32)
    _check((_lib or _library()).llambda_cuda_route(
        desc, logits.ctypes.data, bias.ctypes.data if bias is not None else None, T,
        selected.ctypes.data, weights.ctypes.data))
    return selected, weights


# ------------------------------------------------------------------ 8-bit floating point


def fp8_quantize(x, *, stream=None):
    """(q, scales) of x [T, cols] (float32 or bfloat16): q float8_e4m3fn
    [T, cols rounded up to 16] with zeros past cols, scales float32
    [ceil(cols / 128), T rounded up to 4] with zeros past T, so that x[t, c] is
    about q[t, c] * scales[c // 128, t].  scale = max(max|x| / 448, 2^-126) of
    the row's block, q = e4m3(x / scale), everything rounded to nearest."""
    T, cols, ldx = _matrix(x, "x")
    dev = x.device
    raw, (q, scales) = _on(stream, dev, (x,), lambda: (
        _t.empty((T, _pad(cols, 16)), dtype=_t.float8_e4m3fn, device=dev),
        _t.empty((_blocks(cols), _pad(T, 4)), dtype=_t.float32, device=dev)))
    _check((_lib or _library()).llambda_cuda_fp8_quantize_device(
        _tag(x.dtype), x.data_ptr(), ldx, T, cols, q.data_ptr(), scales.data_ptr(), raw))
    return q, scales


def _device_weights(pair, name: str, ndim: int, device=None):
    """Checks (weights, scales) in device memory."""
    torch = _torch()
    w, s = pair
    _device_tensor(w, f"{name} weights", (torch.float8_e4m3fn, torch.uint8), (None,) * ndim, device,
                   contiguous=True)
    want = tuple(w.shape[:-2]) + (_blocks(w.shape[-2]), _blocks(w.shape[-1]))
    _device_tensor(s, f"{name} scales", (torch.float32,), want, w.device, contiguous=True)
    return w, s


def _host_weights(pair, name: str, ndim: int):
    w, s = pair
    w = np.ascontiguousarray(w)
    if w.dtype.itemsize != 1 or w.ndim != ndim or 0 in w.shape:
        raise ValueError(f"{name} weights must be e4m3 bytes with {ndim} axes")
    w = w.view(np.uint8)
    s = N._f32(s)
    want = w.shape[:-2] + (_blocks(w.shape[-2]), _blocks(w.shape[-1]))
    if s.shape != want:
        raise ValueError(f"{name} scales have shape {s.shape}, expected {want}")
    return w, s


def _fp8_tensor(shape, data: int, scales: int):
    ne2 = shape[0] if len(shape) == 3 else 1
    return N.Fp8Tensor(shape[-1], shape[-2], ne2, data, scales)


class _Fp8Session:
    """What both kinds of session share: the handle and the memory it borrows."""
    _destroy = _status = ""

    def status(self) -> int:
        """Waits for the device; its status word, cleared by reading: 0, or 2
        after a wait inside a kernel timed out."""
        rc = getattr(N.lib(), self._status)(self._h)
        if rc < 0:
            raise N.LlambdaCudaError(N.last_error())
        return rc

    def close(self) -> None:
        if getattr(self, "_h", None):
            getattr(N.lib(), self._destroy)(self._h)
            self._h = None
        self._keep = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _handle(self):
        if not self._h:
            raise ValueError("the session is closed")
        return self._h


class Fp8ProjectionSession(_Fp8Session):
    """One e4m3 matrix [rows][cols] with a scale per 128 x 128 block, resident on
    the GPU: run* returns x . W^T."""
    _destroy = "llambda_cuda_fp8_session_destroy"
    _status = "llambda_cuda_fp8_session_status"

    def __init__(self, handle, rows: int, cols: int, device=None, keep=None):
        self._h, self._keep = handle, keep
        self.rows, self.cols, self.device = rows, cols, device

    @classmethod
    def _create(cls, w, s, data, scales, on_device, device, keep):
        h = C.c_void_p()
        t = _fp8_tensor(w.shape, data, scales)
        _check((_lib or _library()).llambda_cuda_fp8_session_create(
            C.byref(t), on_device, C.byref(h)))
        return cls(h, w.shape[0], w.shape[1], device, keep)

    @classmethod
    def from_tensor(cls, weights, scales):
        """Copies host arrays: weights [rows][cols] of e4m3 bytes, scales
        [ceil(rows / 128)][ceil(cols / 128)] float32."""
        w, s = _host_weights((weights, scales), "projection", 2)
        return cls._create(w, s, w.ctypes.data, s.ctypes.data, 0, None, None)

    @classmethod
    def from_device(cls, weights, scales):
        """Borrows CUDA tensors (kept alive by the session): weights
        float8_e4m3fn or uint8, cols a multiple of 16.  Waits for the device, so
        whatever stream writes them, the scales are checked when written."""
        w, s = _device_weights((weights, scales), "projection", 2)
        with _torch().cuda.device(w.device):
            return cls._create(w, s, w.data_ptr(), s.data_ptr(), 1, w.device, (w, s))

    def run(self, x: np.ndarray) -> np.ndarray:
        """Host arrays: x [T][cols] (or one vector) -> [T][rows] float32."""
        x = N._f32(x)
        one = x.ndim == 1
        x = x.reshape(1, -1) if one else x
        if x.ndim != 2 or x.shape[1] != self.cols or not x.size:
            raise ValueError(f"x must be [tokens][{self.cols}]")
        out = np.empty((x.shape[0], self.rows), np.float32)
        _check((_lib or _library()).llambda_cuda_fp8_session_run(
            self._handle(), x.ctypes.data, x.shape[0], out.ctypes.data))
        return out[0] if one else out

    def run_device(self, x, out=None, *, out_dtype=None, stream=None):
        """x [T, cols] (float32 or bfloat16 CUDA tensor) -> out [T, rows], made
        of `out_dtype` (default x's) unless given."""
        h = self._handle()
        T, _, ldx = _matrix(x, "x", self.cols, self.device)
        dev = x.device
        nbytes = (_lib or _library()).llambda_cuda_fp8_session_workspace(h, T)
        raw, ((out, ldo), work) = _on(stream, dev, (x, out), lambda: (
            _out(out, T, self.rows, out_dtype or x.dtype, dev),
            _t.empty(nbytes, dtype=_t.uint8, device=dev) if nbytes else None))
        _check((_lib or _library()).llambda_cuda_fp8_session_run_device(
            h, _tag(x.dtype), x.data_ptr(), ldx, T, _tag(out.dtype), out.data_ptr(), ldo,
            work.data_ptr() if nbytes else None, nbytes, raw))
        return out

    def run_quantized(self, q, scales, tokens: int, out=None, *, out_dtype=None, stream=None):
        """As run_device over what fp8_quantize returned for `tokens` rows of
        `cols` columns (several projections of one input quantise it once)."""
        torch = _torch()
        h = self._handle()
        _device_tensor(q, "q", (torch.float8_e4m3fn, torch.uint8), (tokens, _pad(self.cols, 16)),
                       self.device, contiguous=True)
        _device_tensor(scales, "scales", (torch.float32,), (_blocks(self.cols), _pad(tokens, 4)),
                       q.device, contiguous=True)
        raw, (out, ldo) = _on(stream, q.device, (q, scales, out), lambda: _out(
            out, tokens, self.rows, out_dtype or torch.float32, q.device))
        _check((_lib or _library()).llambda_cuda_fp8_session_run_quantized(
            h, q.data_ptr(), scales.data_ptr(), tokens, _tag(out.dtype), out.data_ptr(), ldo, raw))
        return out


class Fp8MoeSession(_Fp8Session):
    """The routed experts of one layer in e4m3: expert e of an input x gives
    down_e . q(h), h = silu(gate_e . x) * (up_e . x), or relu(up_e . x)^2 without
    gate, x and h quantised as by fp8_quantize.  up and gate are [E][I][H], down
    [E][O][I], each a pair (weights, scales [E][ceil(rows/128)][ceil(cols/128)])."""
    _destroy = "llambda_cuda_fp8_moe_session_destroy"
    _status = "llambda_cuda_fp8_moe_session_status"

    def __init__(self, handle, experts: int, hidden: int, out_features: int, device=None,
                 keep=None):
        self._h, self._keep = handle, keep
        self.experts, self.hidden, self.out_features = experts, hidden, out_features
        self.device = device

    @classmethod
    def _create(cls, up, down, gate, ptr, on_device, device):
        ts = [_fp8_tensor(p[0].shape, ptr(p[0]), ptr(p[1])) if p is not None
              else N.Fp8Tensor(0, 0, 0, None, None) for p in (gate, up, down)]
        h = C.c_void_p()
        _check((_lib or _library()).llambda_cuda_fp8_moe_session_create(
            *(C.byref(t) for t in ts), on_device, C.byref(h)))
        E, _, H = up[0].shape
        return cls(h, E, H, down[0].shape[1], device, (up, down, gate) if on_device else None)

    @classmethod
    def from_tensor(cls, up, down, gate=None):
        """Copies host arrays of e4m3 bytes and float32 scales."""
        up, down = _host_weights(up, "up", 3), _host_weights(down, "down", 3)
        gate = _host_weights(gate, "gate", 3) if gate is not None else None
        return cls._create(up, down, gate, lambda a: a.ctypes.data, 0, None)

    @classmethod
    def from_device(cls, up, down, gate=None):
        """Borrows CUDA tensors (kept alive by the session), H and I multiples
        of 16, after waiting for the device."""
        up = _device_weights(up, "up", 3)
        dev = up[0].device
        down = _device_weights(down, "down", 3, dev)
        gate = _device_weights(gate, "gate", 3, dev) if gate is not None else None
        with _torch().cuda.device(dev):
            return cls._create(up, down, gate, lambda t: t.data_ptr(), 1, dev)

    def run(self, x: np.ndarray, selected: np.ndarray, weights: np.ndarray) -> np.ndarray:
        """Host arrays: x [T][H], selected and weights [T][k] -> [T][O] float32."""
        x, weights = N._f32(x), N._f32(weights)
        selected = np.ascontiguousarray(selected, dtype=np.int32)
        if x.ndim != 2 or x.shape[1] != self.hidden or not x.size:
            raise ValueError(f"x must be [tokens][{self.hidden}]")
        if selected.ndim != 2 or selected.shape[0] != x.shape[0] or not selected.size \
                or weights.shape != selected.shape:
            raise ValueError("selected and weights must both be [tokens][k]")
        out = np.empty((x.shape[0], self.out_features), np.float32)
        _check((_lib or _library()).llambda_cuda_fp8_moe_session_run(
            self._handle(), x.ctypes.data, x.shape[0], selected.shape[1], selected.ctypes.data,
            weights.ctypes.data, out.ctypes.data))
        return out

    def run_device(self, x, selected, weights, out=None, *, out_dtype=None, stream=None):
        """x [T, H] (float32 or bfloat16), selected int32 and weights float32
        [T, k] (route_experts' results) -> out [T, O] = the weighted sum over a
        token's entries, made of `out_dtype` (default x's) unless given.  Entries
        whose expert is outside 0..E-1 add nothing."""
        h = self._handle()
        T, _, ldx = _matrix(x, "x", self.hidden, self.device)
        dev = x.device
        k = selected.shape[1] if getattr(selected, "ndim", 0) == 2 else None
        _device_tensor(selected, "selected", _INT, (T, k), dev, contiguous=True)
        _device_tensor(weights, "weights", _F32, (T, k), dev, contiguous=True)
        nbytes = (_lib or _library()).llambda_cuda_fp8_moe_session_workspace(h, T, k)
        raw, ((out, ldo), work) = _on(stream, dev, (x, selected, weights, out), lambda: (
            _out(out, T, self.out_features, out_dtype or x.dtype, dev),
            _t.empty(nbytes, dtype=_t.uint8, device=dev)))
        _check((_lib or _library()).llambda_cuda_fp8_moe_session_run_device(
            h, _tag(x.dtype), x.data_ptr(), ldx, T, k, selected.data_ptr(), weights.data_ptr(),
            _tag(out.dtype), out.data_ptr(), ldo, work.data_ptr(), nbytes, raw))
        return out
