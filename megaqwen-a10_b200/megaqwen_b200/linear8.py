"""Linear layer in 8-bit integers: INT8 weights with a scale for each output channel (what quantize_per_channel
makes) and activations quantised on the fly with a scale for each token (csrc/linear8.cu).

    s_x[m] = max(fp32(max|x[m]| / 127), 1e-12),  c = round half even (x / s_x),  y = (c W^T) s_x[m] s_w[n]

The product is exact (int32 sums), so nothing but the rounding of x to 8 bits and of y to its type is lost.  Up
to four tokens of a small layer run as one kernel; else a kernel quantises the tokens and the tensor cores multiply.  A token that holds an infinity or a
NaN gives a row of NaN.
"""
import ctypes

import torch

from . import _lib
from .kv4 import _DTYPES

_workspaces = {}   # (device index, stream) -> (scratch for the quantised tokens, address, bytes)


class Int8Linear:
    """y = x W^T for weight int8 [N, K] and weight_scale fp32 [N] on one CUDA device.

    Rows that are not 16-byte aligned (K not a multiple of 16, odd strides) are copied once into padded rows; other
    weights are used in place.  K <= 131072.  Calls run on torch's current stream and do not synchronise."""

    def __init__(self, weight, weight_scale):
        if not isinstance(weight, torch.Tensor) or not isinstance(weight_scale, torch.Tensor):
            raise TypeError("Int8Linear: tensors expected")
        if not weight.is_cuda:
            raise ValueError("Int8Linear needs CUDA tensors (no CPU path in this library)")
        if weight.dtype != torch.int8 or weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
            raise ValueError(f"weight: int8 [N, K] expected, got {weight.dtype} {tuple(weight.shape)}")
        if weight.shape[1] > 131072:
            raise ValueError("K must be at most 131072 (the sum is 32-bit)")
        if weight_scale.dtype != torch.float32 or weight_scale.shape != (weight.shape[0],) or weight_scale.device != weight.device:
            raise ValueError(f"weight_scale: fp32 [{weight.shape[0]}] on {weight.device} expected")
        n, k = weight.shape
        if k % 16 or weight.stride(1) != 1 or weight.stride(0) % 16 or weight.stride(0) < k or weight.data_ptr() % 16:
            padded = torch.zeros((n, (k + 15) // 16 * 16), dtype=torch.int8, device=weight.device)
            padded[:, :k] = weight
            weight = padded[:, :k]
        self.weight, self.weight_scale = weight, weight_scale.contiguous()
        self.in_features, self.out_features = k, n
        self.device = weight.device
        self.status_ = torch.zeros(2, dtype=torch.int32, device=self.device)
        self._fn = _lib.load().mq_linear8
        self._index = self.device.index
        self._fixed = (weight.data_ptr(), weight.stride(0), self.weight_scale.data_ptr(), self.status_.data_ptr())
        torch.cuda.current_stream(self.device).synchronize()   # the copies are done, whatever stream the first call is on

    def __call__(self, x, out_dtype=None):
        """x [..., K] (bf16, fp16 or fp32, contiguous last axis) -> y [..., N] of out_dtype (default: x's type)."""
        if not isinstance(x, torch.Tensor):
            raise TypeError("Int8Linear: expected a tensor")
        if x.device != self.device:
            raise ValueError(f"x: on {x.device}, expected {self.device}")
        if out_dtype is None:
            out_dtype = x.dtype
        dt, odt = _DTYPES.get(x.dtype), _DTYPES.get(out_dtype)
        if dt is None or odt is None:
            raise ValueError(f"x: {x.dtype} to {out_dtype}, expected of {[str(d) for d in _DTYPES]}")
        k, n, shape = self.in_features, self.out_features, x.shape
        if len(shape) < 1 or shape[-1] != k:
            raise ValueError(f"x: shape {tuple(shape)}, expected [..., {k}]")
        if k > 1 and x.stride(-1) != 1:
            raise ValueError("x: the last axis must be contiguous")
        if len(shape) == 2:
            m, rows = shape[0], x
            out = x.new_empty((m, n), dtype=out_dtype)
        else:
            out = x.new_empty((*shape[:-1], n), dtype=out_dtype)
            rows = x.reshape(-1, k)
            m = rows.shape[0]
        if m == 0:
            return out
        if torch.cuda.current_device() != self._index:
            with torch.cuda.device(self.device):
                self._launch(rows, dt, out, odt, m, n, k)
        else:
            self._launch(rows, dt, out, odt, m, n, k)
        return out

    def _launch(self, rows, dt, out, odt, m, n, k):
        stream = torch._C._cuda_getCurrentRawStream(self._index)
        need = (m * ((k + 15) // 16 * 16) + 255) // 256 * 256 + (4 * m + 15) // 16 * 16   # mq_linear8_workspace_bytes
        graph = torch._C._cuda_isCurrentStreamCapturing()
        space = None if graph else _workspaces.get((self._index, stream))
        if space is None or space[2] < need:
            buf = torch.empty(need, dtype=torch.uint8, device=self.device)
            space = buf, buf.data_ptr(), need
            if not graph:   # a graph's scratch is the graph's alone
                _workspaces[self._index, stream] = space
        _, ws, nbytes = space
        w, ldw, scale, status = self._fixed
        rc = self._fn(rows.data_ptr(), dt, rows.stride(0), w, ldw, scale, out.data_ptr(), odt, m, n, k, ws, nbytes, status, stream)
        if rc:
            _lib.check(rc, "mq_linear8")

    def check_device(self):
        """Raises if a bounded wait of a call ran out; synchronises."""
        code, info = self.status_.tolist()
        if code:
            self.status_.zero_()
            raise _lib.MQError(f"Int8Linear: device error {code} ({_lib.MQ_DEV_ERRORS.get(code, '?')}, at {info})")
