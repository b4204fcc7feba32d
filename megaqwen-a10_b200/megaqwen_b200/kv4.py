"""KV cache held in 4 bits, and attention over it (csrc/kv4.cu, csrc/kv4_attend.cu, csrc/kv4_rows.cu).

The decoder classes keep K and V in bf16: 114,688 bytes for each position of the
28-layer model, which bounds how many long sequences fit a GPU.  `KV4Cache` holds
them as 4-bit codes with one bf16 scale for every `group` dims (32,256 bytes at
group 32, 29,568 at group 128):

    s = bf16(max|x| / 7),  code = clamp(round half even (x / s), -7, 7),  value = code * s

`append` quantises the K and V of new tokens as it writes them, `attend` is causal
attention of the newest tokens (one for each sequence, or a chunk) over what the
cache holds, `read` gives values back.  Positions lie in pages; without a page
table every sequence owns a fixed run of pages.

All calls run on torch's current stream and do not synchronise; lengths and
positions stay on the device.  A position or page outside the cache is reported
by `check_device`, as the decoders report theirs.  A quantisation group that holds
an infinity or a NaN reads back as NaN.
"""
import ctypes
import threading

import torch

from . import _lib
from .config import HEAD_DIM, NUM_KV_HEADS

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}   # MQ_BF16, MQ_FP16, MQ_FP32
_QUERY_DTYPES = (torch.bfloat16, torch.float16)
_Strides = ctypes.c_int64 * 3

_capturing = torch._C._cuda_isCurrentStreamCapturing


class MQKV4Cache(ctypes.Structure):
    """Mirror of MQKV4Cache in include/megaqwen_b200.h."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("k_codes", "k_scales", "v_codes", "v_scales", "page_table", "status")] + \
               [(n, ctypes.c_int) for n in ("batch", "pages_per_seq", "num_pages", "page_size", "max_seq_len",
                                            "num_kv_heads", "head_dim", "group")]


class KV4Cache:
    """4-bit KV cache of `batch` sequences of up to max_seq_len positions.

    head_dim 64 or 128; group 32, 64 or 128 (at most head_dim); page_size 16, 32,
    64, 128 or 256; batch <= 4096.  page_table: int32 [batch, pages_per_seq] on the
    device, entries in [0, num_pages) (entries of pages that are not reached yet may
    hold anything); its owner may change it between calls.  Without one, sequence b
    owns pages b * pages_per_seq ...
    """
    def __init__(self, num_layers, batch, max_seq_len, num_kv_heads=NUM_KV_HEADS, head_dim=HEAD_DIM, group=32,
                 page_size=64, page_table=None, num_pages=None, device="cuda"):
        for name, v in (("num_layers", num_layers), ("batch", batch), ("max_seq_len", max_seq_len),
                        ("num_kv_heads", num_kv_heads)):
            if v < 1:
                raise ValueError(f"{name} must be positive")
        if batch > 4096:
            raise ValueError("batch must be at most 4096")
        if head_dim not in (64, 128):
            raise ValueError("head_dim must be 64 or 128")
        if group not in (32, 64, 128) or group > head_dim:
            raise ValueError("group must be 32, 64 or 128 and at most head_dim")
        if page_size not in (16, 32, 64, 128, 256):
            raise ValueError("page_size must be 16, 32, 64, 128 or 256")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("the cache needs a CUDA device (no CPU path in this library)")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        pages = (max_seq_len + page_size - 1) // page_size
        if page_table is not None:
            if not isinstance(page_table, torch.Tensor) or page_table.dtype != torch.int32 or page_table.dim() != 2:
                raise ValueError("page_table: int32 [batch, pages_per_seq] expected")
            if page_table.device != self.device or not page_table.is_contiguous():
                raise ValueError(f"page_table: contiguous on {self.device} expected")
            if page_table.shape[0] != batch or page_table.shape[1] < pages:
                raise ValueError(f"page_table: {tuple(page_table.shape)}, expected [{batch}, >= {pages}]")
            if num_pages is None or num_pages < 1:
                raise ValueError("num_pages is needed with a page_table")
            pages = page_table.shape[1]
        elif num_pages is not None and num_pages < batch * pages:
            raise ValueError(f"num_pages {num_pages}: {batch * pages} needed without a page_table")
        else:
            num_pages = batch * pages if num_pages is None else num_pages
        self.num_layers, self.batch, self.max_seq_len = num_layers, batch, max_seq_len
        self.num_kv_heads, self.head_dim, self.group, self.page_size = num_kv_heads, head_dim, group, page_size
        self.num_pages, self.page_table = num_pages, page_table
        shape = (2, num_layers, num_pages, num_kv_heads, page_size)
        self.codes = torch.full((*shape, head_dim // 2), 0x88, dtype=torch.uint8, device=self.device)   # all values 0
        self.scales = torch.zeros((*shape, head_dim // group), dtype=torch.bfloat16, device=self.device)
        self.status_ = torch.zeros(2, dtype=torch.int32, device=self.device)
        self._lib = _lib.load()
        self._views, self._refs = [], []
        for i in range(num_layers):
            v = MQKV4Cache(self.codes[0, i].data_ptr(), self.scales[0, i].data_ptr(), self.codes[1, i].data_ptr(),
                           self.scales[1, i].data_ptr(), page_table.data_ptr() if page_table is not None else None,
                           self.status_.data_ptr(), batch, pages, num_pages, page_size, max_seq_len, num_kv_heads,
                           head_dim, group)
            self._views.append(v)
            self._refs.append(ctypes.byref(v))
        self._sizes, self._spaces, self._lock = {}, {}, threading.Lock()
        self._seq_shape, self._index, self._scale = torch.Size((batch,)), self.device.index, head_dim ** -0.5
        torch.cuda.current_stream(self.device).synchronize()   # the fills are done, whatever stream the first call is on

    # -- arguments ---------------------------------------------------------
    def _layer(self, layer):
        if not 0 <= layer < self.num_layers:
            raise ValueError(f"layer {layer} outside [0, {self.num_layers})")
        return self._refs[layer]

    def _per_seq(self, x, name):
        if not isinstance(x, torch.Tensor):
            x = torch.as_tensor(x, dtype=torch.int32).to(self.device)
        if x.dtype is not torch.int32 or x.shape != self._seq_shape or x.device != self.device or not x.is_contiguous():
            raise ValueError(f"{name}: contiguous int32 [{self.batch}] on {self.device} expected, "
                             f"got {x.dtype} {tuple(x.shape)} on {x.device}")
        return x

    def _tokens(self, x, name, heads, dtypes):
        """(tokens, heads, strides of the first three axes) of x [batch, tokens, heads, head_dim]; heads: how many, or 0."""
        if not isinstance(x, torch.Tensor):
            raise TypeError(f"{name}: expected a tensor")
        if x.device != self.device:
            raise ValueError(f"{name}: on {x.device}, expected {self.device}")
        if x.dtype not in dtypes:
            raise ValueError(f"{name}: dtype {x.dtype}, expected one of {[str(d) for d in dtypes]}")
        shape = x.shape
        if len(shape) != 4 or shape[0] != self.batch or (heads and shape[2] != heads) or shape[3] != self.head_dim:
            raise ValueError(f"{name}: shape {tuple(shape)}, expected [{self.batch}, tokens, "
                             f"{heads or 'heads'}, {self.head_dim}]")
        sb, st, sh, sd = x.stride()
        if sd != 1:
            raise ValueError(f"{name}: the last axis must be contiguous")
        return shape[1], shape[2], _Strides(sb, st, sh)

    def _call(self, what, fn, *args):
        stream = torch._C._cuda_getCurrentRawStream(self._index)
        if torch.cuda.current_device() != self._index:
            with torch.cuda.device(self.device):
                rc = fn(*args, stream)
        else:
            rc = fn(*args, stream)
        if rc:
            _lib.check(rc, what)

    # -- operators ---------------------------------------------------------
    def append(self, layer, k, v, positions, counts=None):
        """Quantises and writes k and v [batch, tokens, kv heads, head_dim] (bf16, fp16 or fp32, any strides with a
        contiguous last axis): token t of sequence b at position positions[b] + t, for t < counts[b] (default: all).
        positions, counts: int32 [batch] on the device, or lists."""
        ref = self._layer(layer)
        tokens, _, ks = self._tokens(k, "k", self.num_kv_heads, _DTYPES)
        _, _, vs = self._tokens(v, "v", self.num_kv_heads, (k.dtype,))
        if v.shape != k.shape:
            raise ValueError(f"v: shape {tuple(v.shape)}, k has {tuple(k.shape)}")
        positions = self._per_seq(positions, "positions")
        counts = self._per_seq(counts, "counts") if counts is not None else None
        self._call("mq_kv4_append", self._lib.mq_kv4_append, ref, _DTYPES[k.dtype], k.data_ptr(), ks, v.data_ptr(), vs,
                   positions.data_ptr(), counts.data_ptr() if counts is not None else None, tokens)

    def read(self, layer, starts, n, dtype=torch.bfloat16):
        """The values of positions starts[b] .. starts[b] + n - 1: (k, v), each [batch, kv heads, n, head_dim] -- the
        decoders' cache layout.  Positions outside [0, max_seq_len) are zeros."""
        ref = self._layer(layer)
        if dtype not in _DTYPES:
            raise ValueError(f"dtype {dtype}, expected one of {[str(d) for d in _DTYPES]}")
        if n < 0:
            raise ValueError("n must not be negative")
        starts = self._per_seq(starts, "starts")
        k, v = self.scales.new_empty((2, self.batch, self.num_kv_heads, n, self.head_dim), dtype=dtype).unbind(0)
        self._call("mq_kv4_read", self._lib.mq_kv4_read, ref, starts.data_ptr(), n, _DTYPES[dtype], k.data_ptr(), v.data_ptr())
        return k, v

    def attend(self, layer, q, lengths, counts=None, scale=None):
        """Causal attention of q [batch, tokens, q heads, head_dim] (bf16 or fp16) over the cache, which already holds
        the new tokens: lengths[b] positions in all, the last counts[b] (default: tokens) of them the rows of q.  Rows
        t >= counts[b] are padding, and give zeros as rows before position 0 do.  scale: default head_dim ** -0.5.
        Returns a new contiguous tensor like q."""
        ref = self._layer(layer)
        tokens, heads, qs = self._tokens(q, "q", 0, _QUERY_DTYPES)
        if heads < 1 or heads % self.num_kv_heads:
            raise ValueError(f"q: {heads} heads, expected a multiple of {self.num_kv_heads}")
        lengths = self._per_seq(lengths, "lengths")
        counts = self._per_seq(counts, "counts") if counts is not None else None
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        if tokens == 0:
            return out
        space, _alive = self._space(ref, tokens, heads)
        self._call("mq_kv4_attend", self._lib.mq_kv4_attend, ref, _DTYPES[q.dtype], q.data_ptr(), qs, out.data_ptr(),
                   lengths.data_ptr(), counts.data_ptr() if counts is not None else None, tokens, heads,
                   self._scale if scale is None else float(scale), *space)
        return out

    def _space(self, ref, tokens, heads):
        """((scratch, bytes, counters, number), tensors) for a call on the current stream: each stream has its own, and so
        has each call that a graph captures (the graph zeroes its counters), so calls and graphs may overlap on different
        streams."""
        key, graph = torch._C._cuda_getCurrentRawStream(self._index), _capturing()
        args = self._sizes.get((key, tokens, heads))
        if args is None or graph:
            nbytes, ncnt = ctypes.c_size_t(0), ctypes.c_size_t(0)
            with self._lock, torch.cuda.device(self.device):
                _lib.check(self._lib.mq_kv4_attend_workspace(ref, tokens, heads, ctypes.byref(nbytes), ctypes.byref(ncnt)),
                           "mq_kv4_attend_workspace")
                have = None if graph else self._spaces.get(key)
                if have is None or have[0].numel() < nbytes.value or have[1].numel() < ncnt.value:
                    have = (torch.empty(nbytes.value, dtype=torch.uint8, device=self.device),
                            torch.zeros(ncnt.value, dtype=torch.int32, device=self.device))
                    if not graph:
                        self._spaces[key] = have
                        for other in [k for k in list(self._sizes) if k[0] == key]:   # they hold the old one's address
                            del self._sizes[other]
                args = (have[0].data_ptr(), have[0].numel(), have[1].data_ptr(), have[1].numel()), have
                if not graph:
                    self._sizes[key, tokens, heads] = args
        return args

    def status(self):
        """(code, sequence) of the device-side status word (MQ_DEV_*); synchronises."""
        return tuple(self.status_.tolist())

    def check_device(self):
        """Raises (and clears the status) if a call met a position or a page outside the cache."""
        code, info = self.status()
        if code:
            self.status_.zero_()
            raise _lib.MQError(f"4-bit cache: device error {code} ({_lib.MQ_DEV_ERRORS.get(code, '?')}, sequence {info})")
