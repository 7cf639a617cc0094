"""Python-side mirror of the operator interface: torch (or raw pointers) in, C ABI underneath.

torch is used only for device memory and the current CUDA stream; every operator call goes to
``libko_b200.so``.  ``Tensor`` mirrors the reference's ``class Tensor`` (common/tensor.h:11-40):
a page-locked host buffer plus a device buffer with copies in both directions.
"""
from __future__ import annotations

import ctypes as C
import functools

import numpy as np

from . import native

DTYPE_F32, DTYPE_F16, DTYPE_BF16 = 0, 1, 2
_NP_OF = {DTYPE_F32: np.float32, DTYPE_F16: np.uint16, DTYPE_BF16: np.uint16}
_SIZE_OF = {DTYPE_F32: 4, DTYPE_F16: 2, DTYPE_BF16: 2}


def _current_stream_ptr(device_index: int | None = None) -> int:
    """Handle of the current stream of a device (None: the current one).  The handle alone: building the Stream object
    around it (torch.cuda.current_stream()) costs the host 3 us a call."""
    import torch

    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if device_index is None else device_index)


def _ptr(t) -> int | None:
    """Device address of a torch tensor (must be contiguous), an int address, or None."""
    if t is None:
        return None
    if isinstance(t, int):
        return t
    if not t.is_cuda:
        raise ValueError("operator inputs must live on a CUDA device (there is no CPU path)")
    if not t.is_contiguous():
        raise ValueError("operator inputs must be contiguous")
    return int(t.data_ptr())


class Tensor:
    """Host (pinned) + device buffer of ``size_in_bytes`` bytes owned by the native library."""

    def __init__(self, size_in_bytes: int, device: int = -1):
        self._h = C.c_void_p()
        native.check(native.lib().ko_tensor_create(size_in_bytes, device, C.byref(self._h)), "ko_tensor_create")

    @classmethod
    def from_shape(cls, shape, byte_per_element: int, device: int = -1) -> "Tensor":
        return cls(int(np.prod(shape, dtype=np.int64)) * byte_per_element, device)

    def __del__(self):
        try:
            self.close()
        except Exception:  # interpreter shutdown: the module globals are already gone, the process frees the buffers
            pass

    def close(self) -> None:
        if getattr(self, "_h", None) is not None and self._h.value:
            native.lib().ko_tensor_destroy(self._h)
            self._h = C.c_void_p()

    @property
    def size_in_bytes(self) -> int:
        return int(native.lib().ko_tensor_size_in_bytes(self._h))

    @property
    def device(self) -> int:
        return int(native.lib().ko_tensor_device(self._h))

    @property
    def device_ptr(self) -> int:
        return int(native.lib().ko_tensor_device_ptr(self._h) or 0)

    def host_ref(self, dtype=np.float32) -> np.ndarray:
        """numpy view of the host buffer (no copy)."""
        n = self.size_in_bytes // np.dtype(dtype).itemsize
        addr = native.lib().ko_tensor_host_ptr(self._h)
        buf = (C.c_char * self.size_in_bytes).from_address(addr)
        return np.frombuffer(buf, dtype=dtype, count=n)

    def host_to_device(self) -> None:
        native.check(native.lib().ko_tensor_host_to_device(self._h), "ko_tensor_host_to_device")

    def host_to_device_async(self, stream: int | None = None) -> None:
        s = _current_stream_ptr() if stream is None else stream
        native.check(native.lib().ko_tensor_host_to_device_async(self._h, s), "ko_tensor_host_to_device_async")

    def device_to_host(self) -> None:
        native.check(native.lib().ko_tensor_device_to_host(self._h), "ko_tensor_device_to_host")

    def device_to_host_async(self, stream: int | None = None) -> None:
        s = _current_stream_ptr() if stream is None else stream
        native.check(native.lib().ko_tensor_device_to_host_async(self._h, s), "ko_tensor_device_to_host_async")


# ------------------------------------------------------------------ seeded host fills
def fill_uniform(shape, seed: int, tensor_id: int, lo=-1.0, hi=1.0, dtype: int = DTYPE_F32, elem_offset: int = 0,
                 out: np.ndarray | None = None) -> np.ndarray:
    a = np.empty(shape, dtype=_NP_OF[dtype]) if out is None else out
    native.check(native.lib().ko_fill_uniform(a.ctypes.data, dtype, a.size, seed, tensor_id, elem_offset, lo, hi),
                 "ko_fill_uniform")
    return a


def fill_normal(shape, seed: int, tensor_id: int, mean=0.0, std=1.0, dtype: int = DTYPE_F32, elem_offset: int = 0,
                out: np.ndarray | None = None) -> np.ndarray:
    a = np.empty(shape, dtype=_NP_OF[dtype]) if out is None else out
    native.check(native.lib().ko_fill_normal(a.ctypes.data, dtype, a.size, seed, tensor_id, elem_offset, mean, std),
                 "ko_fill_normal")
    return a


def fill_causal_mask_(a: np.ndarray, row_offset: int = 0, block: int = 512, value: float = -1e4) -> np.ndarray:
    rows, cols = a.shape
    assert a.dtype == np.float32 and a.flags["C_CONTIGUOUS"]
    native.check(native.lib().ko_fill_causal_mask_f32(a.ctypes.data, rows, cols, row_offset, block, value),
                 "ko_fill_causal_mask_f32")
    return a


# ------------------------------------------------------------------ operators (torch tensors on the GPU)
def softmax(x, out=None, stream: int | None = None):
    """Row softmax over the last dimension of a 2-D FP32, FP16 or BF16 CUDA tensor (FP32 arithmetic)."""
    import torch

    assert x.dim() == 2 and x.dtype in (torch.float32, torch.float16, torch.bfloat16)
    out = torch.empty_like(x) if out is None else out
    assert out.dtype == x.dtype
    s = _current_stream_ptr() if stream is None else stream
    rows, cols = x.shape
    lib = native.lib()
    fn = {torch.float32: lib.ko_softmax_f32, torch.float16: lib.ko_softmax_f16, torch.bfloat16: lib.ko_softmax_bf16}[x.dtype]
    native.check(fn(_ptr(x), _ptr(out), rows, cols, s), "ko_softmax")
    return out


def layernorm(x, eps: float, gamma=None, beta=None, ddof: int = 0, out=None, stream: int | None = None):
    """LayerNorm forward over the last dimension of a 2-D FP32, FP16 or BF16 CUDA tensor (FP32 statistics)."""
    import torch

    assert x.dim() == 2 and x.dtype in (torch.float32, torch.float16, torch.bfloat16)
    for p in (gamma, beta):
        assert p is None or (p.dtype == x.dtype and p.numel() == x.shape[1])
    out = torch.empty_like(x) if out is None else out
    s = _current_stream_ptr() if stream is None else stream
    rows, cols = x.shape
    lib = native.lib()
    fn = {torch.float32: lib.ko_layernorm_f32, torch.float16: lib.ko_layernorm_f16, torch.bfloat16: lib.ko_layernorm_bf16}[x.dtype]
    native.check(fn(_ptr(x), _ptr(out), rows, cols, eps, _ptr(gamma), _ptr(beta), ddof, s), "ko_layernorm")
    return out


def _operand(t, name: str, device, dtypes, shape) -> int | None:
    """Address of an operand after checking where it lives, its type, shape and layout (None stays None)."""
    if t is None:
        return None
    if t.device == device and t.dtype in dtypes and t.shape == shape and t.is_contiguous():
        return t.data_ptr()
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the operator's first input on {device}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} is {t.dtype}, expected {' or '.join(str(d) for d in dtypes)}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")
    raise ValueError(f"{name} must be contiguous")


def _elsewhere(device, stream: int | None):
    """None when `device` is the current one and `stream` is not given; else a context in which `device` and the stream with
    handle `stream` (None: the device's current one) are current, so that outputs and workspaces come from the pool of the
    stream that uses them."""
    import torch

    if device.type != "cuda":
        raise ValueError("operator inputs must live on a CUDA device (there is no CPU path)")
    if stream is None:
        return None if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)
    if stream == 0:
        return torch.cuda.stream(torch.cuda.default_stream(device))
    return torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device))


def _workspace(nbytes: int, device):
    """(tensor, address, bytes) of device memory for one call: allocated on the current stream, so the caching allocator hands
    it out again only to work that runs after the call (inside a capture: it belongs to the graph)."""
    import torch

    if nbytes == 0:
        return None, None, 0
    t = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return t, t.data_ptr(), nbytes


@functools.lru_cache(maxsize=4096)
def _layernorm_backward_bytes(device_index: int, dtype: int, rows: int, cols: int) -> int:
    n = C.c_size_t()
    native.check(native.lib().ko_layernorm_backward_workspace(dtype, rows, cols, C.byref(n)), "ko_layernorm_backward_workspace")
    return n.value


def layernorm_backward(dy, x, eps: float, gamma=None, ddof: int = 0, residual=None, dx=None, dgamma=None, dbeta=None,
                       stream: int | None = None):
    """Gradients of :func:`layernorm` (same ``eps`` and ``ddof``): ``(dx, dgamma, dbeta)``.

    ``dy``, ``x`` and ``residual`` are 2-D FP32, FP16 or BF16 CUDA tensors of one shape and type, ``gamma`` a vector of that
    type (None: 1).  The statistics are formed again from ``x``.  ``residual`` is the gradient that reaches ``x`` past the norm
    (the skip connection of a pre-norm block) and is added to ``dx``.  ``dx`` has the inputs' type and may be ``dy``, ``x`` or
    ``residual`` itself; ``dgamma`` and ``dbeta`` are FP32.
    """
    import torch

    if x.dim() != 2 or x.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError(f"x must be a 2-D FP32, FP16 or BF16 tensor, got {x.dtype} with {x.dim()} dimensions")
    rows, cols = x.shape
    device, same, vector = x.device, (x.dtype,), (torch.float32,)
    lib = native.lib()
    code, fn = {torch.float32: (DTYPE_F32, lib.ko_layernorm_backward_f32), torch.float16: (DTYPE_F16, lib.ko_layernorm_backward_f16),
                torch.bfloat16: (DTYPE_BF16, lib.ko_layernorm_backward_bf16)}[x.dtype]
    place = _elsewhere(device, stream)
    if place is not None:
        with place:
            return layernorm_backward(dy, x, eps, gamma, ddof, residual, dx, dgamma, dbeta)
    matrix, row = (rows, cols), (cols,)
    x_at, dy_at = _ptr(x), _operand(dy, "dy", device, same, matrix)
    gamma_at, residual_at = _operand(gamma, "gamma", device, same, row), _operand(residual, "residual", device, same, matrix)
    dx_at, dgamma_at, dbeta_at = (_operand(dx, "dx", device, same, matrix), _operand(dgamma, "dgamma", device, vector, row),
                                  _operand(dbeta, "dbeta", device, vector, row))
    if dx is None:
        dx = torch.empty(rows, cols, dtype=x.dtype, device=device)
        dx_at = dx.data_ptr()
    if dgamma is None:
        dgamma = torch.empty(cols, dtype=torch.float32, device=device)
        dgamma_at = dgamma.data_ptr()
    if dbeta is None:
        dbeta = torch.empty(cols, dtype=torch.float32, device=device)
        dbeta_at = dbeta.data_ptr()
    ws, ws_at, ws_bytes = _workspace(_layernorm_backward_bytes(device.index, code, rows, cols), device)
    native.check(fn(dy_at, x_at, dx_at, rows, cols, eps, gamma_at, residual_at, dgamma_at, dbeta_at, ddof, ws_at, ws_bytes,
                    _current_stream_ptr(device.index)), "ko_layernorm_backward")
    return dx, dgamma, dbeta


def softmax_host(t_in: Tensor, t_out: Tensor, rows: int, cols: int, chunks: int = 0, stream: int | None = None) -> None:
    """FP32 row softmax of the HOST contents of ``t_in`` into the host buffer of ``t_out``: copy in, kernel and
    copy out are pipelined over ``chunks`` row ranges (0 = 8).  Stream-ordered like a kernel launch."""
    s = _current_stream_ptr() if stream is None else stream
    native.check(native.lib().ko_softmax_f32_host(t_in._h, t_out._h, rows, cols, chunks, s), "ko_softmax_f32_host")


def layernorm_host(t_in: Tensor, t_out: Tensor, rows: int, cols: int, eps: float, gamma=None, beta=None, ddof: int = 0,
                   chunks: int = 0, stream: int | None = None) -> None:
    """FP32 LayerNorm of the HOST contents of ``t_in`` into the host buffer of ``t_out`` (gamma / beta: CUDA tensors)."""
    s = _current_stream_ptr() if stream is None else stream
    native.check(native.lib().ko_layernorm_f32_host(t_in._h, t_out._h, rows, cols, eps, _ptr(gamma), _ptr(beta), ddof, chunks, s),
                 "ko_layernorm_f32_host")


def sgemm(a, b, c=None, out=None, stream: int | None = None):
    """D = A @ B (+ C); row-major FP32 CUDA tensors."""
    import torch

    assert a.dtype == b.dtype == torch.float32 and a.dim() == b.dim() == 2 and a.shape[1] == b.shape[0]
    M, K = a.shape
    N = b.shape[1]
    out = torch.empty((M, N), dtype=torch.float32, device=a.device) if out is None else out
    s = _current_stream_ptr() if stream is None else stream
    native.check(native.lib().ko_sgemm_f32(M, N, K, _ptr(a), _ptr(b), _ptr(c), _ptr(out), s), "ko_sgemm_f32")
    return out


def gemm_tc(a, b, c=None, out=None, stream: int | None = None, out_dtype=None, b_row_major: bool = False):
    """D[M,N] = A[M,K] @ B[K,N] (+ C) with FP16/BF16 inputs and FP32 accumulation.

    ``b`` is the column-major [K,N] operand as stored, i.e. a contiguous [N,K] tensor, or with
    ``b_row_major`` a contiguous [K,N] tensor.  ``out_dtype`` is float32 (default) or the input dtype;
    ``c`` has the output dtype.
    """
    import torch

    assert a.dtype == b.dtype and a.dtype in (torch.float16, torch.bfloat16)
    M, K = a.shape
    if b_row_major:
        K2, N = b.shape
    else:
        N, K2 = b.shape
    assert K == K2
    out_dtype = (out.dtype if out is not None else torch.float32) if out_dtype is None else out_dtype
    assert out_dtype in (torch.float32, a.dtype), "D is FP32 or the input type"
    assert c is None or c.dtype == out_dtype
    out = torch.empty((M, N), dtype=out_dtype, device=a.device) if out is None else out
    assert out.dtype == out_dtype
    s = _current_stream_ptr() if stream is None else stream
    in_fmt = 0 if a.dtype == torch.float16 else 1
    out_fmt = 0 if out_dtype == torch.float32 else (1 if out_dtype == torch.float16 else 2)
    native.check(native.lib().ko_gemm_tc(in_fmt, out_fmt, 1 if b_row_major else 0, M, N, K, _ptr(a), _ptr(b), _ptr(c), _ptr(out), s),
                 "ko_gemm_tc")
    return out


# ------------------------------------------------------------------ linear layer, forward and backward
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


def _activation_code(name: str) -> int:
    if name not in ACTIVATIONS:
        raise ValueError(f"unknown activation {name!r}, expected one of {', '.join(ACTIVATIONS)}")
    return ACTIVATIONS[name]


def _linear_types(a, out, out_dtype, default):
    """(in_fmt, out_fmt, out_dtype) of a product whose inputs have `a`'s type."""
    import torch

    dtype = a.dtype
    if a.dim() != 2 or (dtype is not torch.bfloat16 and dtype is not torch.float16):
        raise ValueError(f"the inputs must be 2-D FP16 or BF16 tensors, got {dtype} with {a.dim()} dimensions")
    if out_dtype is None:
        out_dtype = default if out is None else out.dtype
    in_fmt = 0 if dtype is torch.float16 else 1
    if out_dtype is dtype:
        return in_fmt, in_fmt + 1, out_dtype
    if out_dtype is not torch.float32:
        raise ValueError(f"the output is FP32 or the inputs' {dtype}, not {out_dtype}")
    return in_fmt, 0, out_dtype


@functools.lru_cache(maxsize=4096)
def _linear_bytes(device_index: int, entry: str, m: int, n: int, k: int) -> int:
    nbytes = C.c_size_t()
    native.check(getattr(native.lib(), entry)(m, n, k, C.byref(nbytes)), entry)
    return nbytes.value


def linear(x, w, bias=None, activation: str = "none", residual=None, out=None, out_dtype=None, return_pre: bool = False, pre=None,
           stream: int | None = None):
    """``y = act(x @ w.T + bias) + residual`` on the tensor cores.

    ``x`` [tokens, k] and ``w`` [n, k] are FP16 or BF16 with k a multiple of 8, ``bias`` [n] has their type; ``y`` and ``residual``
    [tokens, n] have ``out_dtype``: the inputs' type (default) or FP32.  ``activation``: none, relu, gelu (erf), gelu_tanh or silu.
    With ``return_pre`` (or a tensor ``pre`` to write) the result is ``(y, pre)``, ``pre = x @ w.T + bias`` in the inputs' type:
    what :func:`linear_backward_input` of the next layer takes.  ``out`` may be ``residual`` itself.
    """
    import torch

    in_fmt, out_fmt, out_dtype = _linear_types(x, out, out_dtype, x.dtype)
    act = _activation_code(activation)
    device, same, to = x.device, (x.dtype,), (out_dtype,)
    if w.dim() != 2:
        raise ValueError(f"w must have 2 dimensions, got {w.dim()}")
    (m, k), n = x.shape, w.shape[0]
    place = _elsewhere(device, stream)
    if place is not None:
        with place:
            return linear(x, w, bias, activation, residual, out, out_dtype, return_pre, pre)
    matrix = (m, n)
    x_at, w_at, bias_at = _ptr(x), _operand(w, "w", device, same, (n, k)), _operand(bias, "bias", device, same, (n,))
    residual_at, out_at, pre_at = (_operand(residual, "residual", device, to, matrix), _operand(out, "out", device, to, matrix),
                                   _operand(pre, "pre", device, same, matrix))
    if out is None:
        out = torch.empty(m, n, dtype=out_dtype, device=device)
        out_at = out.data_ptr()
    if return_pre and pre is None:
        pre = torch.empty(m, n, dtype=x.dtype, device=device)
        pre_at = pre.data_ptr()
    ws, ws_at, ws_bytes = _workspace(_linear_bytes(device.index, "ko_linear_workspace", m, n, k), device)
    native.check(native.lib().ko_linear(in_fmt, out_fmt, act, m, n, k, x_at, w_at, bias_at, residual_at, out_at, pre_at, ws_at, ws_bytes,
                                        _current_stream_ptr(device.index)), "ko_linear")
    return out if pre is None else (out, pre)


def linear_backward_input(dy, w, pre=None, activation: str = "none", out=None, out_dtype=None, stream: int | None = None):
    """``dx = (dy @ w) * act'(pre)``: the gradient of :func:`linear`'s input, taken on through the activation that made it.

    ``dy`` [tokens, n] and ``w`` [n, k] are FP16 or BF16, n and k multiples of 8; ``pre`` [tokens, k] (the inputs' type) is the
    pre-activation of the layer before, needed unless ``activation`` is none.  ``dx`` [tokens, k] has ``out_dtype``: the inputs'
    type (default; ``out`` may then be ``pre`` itself) or FP32.
    """
    import torch

    in_fmt, out_fmt, out_dtype = _linear_types(dy, out, out_dtype, dy.dtype)
    act = _activation_code(activation)
    device, same = dy.device, (dy.dtype,)
    if w.dim() != 2:
        raise ValueError(f"w must have 2 dimensions, got {w.dim()}")
    (m, n), k = dy.shape, w.shape[1]
    place = _elsewhere(device, stream)
    if place is not None:
        with place:
            return linear_backward_input(dy, w, pre, activation, out, out_dtype)
    dy_at, w_at, pre_at = _ptr(dy), _operand(w, "w", device, same, (n, k)), _operand(pre, "pre", device, same, (m, k))
    out_at = _operand(out, "out", device, (out_dtype,), (m, k))
    if out is None:
        out = torch.empty(m, k, dtype=out_dtype, device=device)
        out_at = out.data_ptr()
    ws, ws_at, ws_bytes = _workspace(_linear_bytes(device.index, "ko_linear_backward_input_workspace", m, n, k), device)
    native.check(native.lib().ko_linear_backward_input(in_fmt, out_fmt, act, m, n, k, dy_at, w_at, pre_at, out_at, ws_at, ws_bytes,
                                                       _current_stream_ptr(device.index)), "ko_linear_backward_input")
    return out


def linear_backward_weight(dy, x, c=None, out=None, out_dtype=None, return_bias: bool = True, dbias=None, stream: int | None = None):
    """``dw = dy.T @ x (+ c)`` and, with ``return_bias`` (or a tensor ``dbias`` to write), ``dbias`` = the column sums of ``dy``.

    ``dy`` [tokens, n] and ``x`` [tokens, k] are FP16 or BF16, n and k multiples of 8, any number of tokens.  ``dw`` and ``c`` [n, k]
    have ``out_dtype``: FP32 (default) or the inputs' type; ``out`` may be ``c`` itself (gradients gathered over micro-batches).
    ``dbias`` [n] is FP32.  Returns ``(dw, dbias)``, or ``dw`` alone.
    """
    import torch

    in_fmt, out_fmt, out_dtype = _linear_types(dy, out, out_dtype, torch.float32)
    device, to = dy.device, (out_dtype,)
    if x.dim() != 2:
        raise ValueError(f"x must have 2 dimensions, got {x.dim()}")
    (m, n), k = dy.shape, x.shape[1]
    place = _elsewhere(device, stream)
    if place is not None:
        with place:
            return linear_backward_weight(dy, x, c, out, out_dtype, return_bias, dbias)
    dy_at, x_at, c_at = _ptr(dy), _operand(x, "x", device, (dy.dtype,), (m, k)), _operand(c, "c", device, to, (n, k))
    out_at, dbias_at = _operand(out, "out", device, to, (n, k)), _operand(dbias, "dbias", device, (torch.float32,), (n,))
    if out is None:
        out = torch.empty(n, k, dtype=out_dtype, device=device)
        out_at = out.data_ptr()
    if return_bias and dbias is None:
        dbias = torch.empty(n, dtype=torch.float32, device=device)
        dbias_at = dbias.data_ptr()
    ws, ws_at, ws_bytes = _workspace(_linear_bytes(device.index, "ko_linear_backward_weight_workspace", m, n, k), device)
    native.check(native.lib().ko_linear_backward_weight(in_fmt, out_fmt, m, n, k, dy_at, x_at, c_at, out_at, dbias_at, ws_at, ws_bytes,
                                                        _current_stream_ptr(device.index)), "ko_linear_backward_weight")
    return out if dbias is None else (out, dbias)
