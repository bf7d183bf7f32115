"""Operators on torch CUDA tensors, beside the embedding model: attention of causal prompts and of texts
behind a shared prefix, and products of a few rows with 4-bit weights.

They need no model and keep nothing between calls (the entry points are ge_attention_causal,
ge_attention_prefix and ge_linear_q4 of include/gemma_embed.h).  Every call enqueues its work on
`stream` -- a torch stream, a raw cudaStream_t, or None for torch's current stream of the
tensors' device -- and returns without synchronising; it may be captured into a CUDA graph.  A stream
other than the current one has to be behind the work that fills the inputs; their memory is not reused
before the call's work there has ended.  A wait inside the attention kernels that ran out (2 s and more,
which no argument can bring about) leaves NaN in the rows it kept from being finished.  There is no
derivative: inputs that require a gradient are refused while gradients are recorded, dual tensors of
forward-mode differentiation always.

    out = attention_causal(q, k, v, seqs)               # q [T, H, D], k and v [T, KV, D]
    last = attention_prefix(q, k, v, q_seqs, kv_seqs, prefix_k, prefix_v)
    y = linear_q4(x, Q4Weight.from_blocks(gguf_bytes, "Q4_0", n, k, device))
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import math
from dataclasses import dataclass
from typing import Any, Optional

import numpy as np

from . import _lib

__all__ = ["attention_causal", "attention_prefix", "linear_q4", "Q4Weight"]

_HERE = contextlib.nullcontext()
# What the entry points take, checked here where a larger number would reach them as its lowest 32 bits.
MAX_ROWS, MAX_HEADS, MAX_SEQUENCES, MAX_WINDOW = 1 << 30, 65535, 1 << 30, (1 << 31) - 1
Q4_MAX_ROWS, Q4_MAX_N, Q4_MAX_K = 64, 1 << 30, 65536
Q4_TYPES = {"Q4_0": 2, "Q4_1": 3}  # GGUF tensor type ids (ge_q4_type)


def _error(code: int, message: str):
    from . import GemmaEmbedError
    return GemmaEmbedError(code, message)


def _invalid(message: str):
    return _error(9, f"invalid options: {message}")


def _call(rc: int):
    if rc != 0:
        raise _error(rc, (_lib.lib().ge_last_error(None) or b"").decode())


@functools.cache
def _torch():
    import torch
    # The current stream's handle without building a torch.cuda.Stream (a microsecond of every call).
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda d: torch.cuda.current_stream(d).cuda_stream)
    return torch, {torch.float16: 0, torch.bfloat16: 1}, raw


@functools.cache
def _forward_ad():
    from torch.autograd import forward_ad
    return forward_ad


def _dtype(t) -> int:
    code = _torch()[1].get(t.dtype)
    if code is None:
        raise _invalid(f"tensors must be float16 or bfloat16, got {t.dtype}")
    return code


def _on_device(name: str, t, device: Optional[int] = None) -> int:
    """The ordinal of the CUDA device that holds `t` (and has to be `device`, when given)."""
    if not isinstance(t, _torch()[0].Tensor) or not t.is_cuda:
        raise _invalid(f"{name} must be a CUDA tensor")
    d = t.get_device()
    if device is not None and d != device:
        raise _invalid(f"{name} is on cuda:{d}, not on cuda:{device}")
    return d


def _no_gradient(name: str, t):
    if t.requires_grad and _torch()[0].is_grad_enabled():
        raise _invalid(f"{name} requires a gradient, and the operator has no backward pass (call it under torch.no_grad())")
    # Inside a forward-mode level (a dual tensor's tangent is not seen from outside).
    forward = _forward_ad()
    if forward._current_level >= 0 and forward.unpack_dual(t).tangent is not None:
        raise _invalid(f"{name} carries a forward-mode tangent, and the operator has no derivative")


def _heads(name: str, t, device: int, dtype, heads: Optional[int], dim: int):
    """Checks a [rows, heads, dim] tensor; gives its rows, heads and the elements between its rows."""
    _on_device(name, t, device)
    if t.dtype != dtype:
        raise _invalid(f"{name} is {t.dtype}, not {dtype}")
    _no_gradient(name, t)
    shape = t.shape
    if len(shape) != 3 or shape[2] != dim or (heads is not None and shape[1] != heads):
        want = f"[rows, {heads if heads is not None else 'heads'}, {dim}]"
        raise _invalid(f"{name} must be {want}, got {list(shape)}")
    rows, n, _ = shape
    if rows > MAX_ROWS or n > MAX_HEADS:
        raise _invalid(f"{name} must have at most 2^30 rows and {MAX_HEADS} heads, got {list(shape)}")
    s0, s1, s2 = t.stride()
    if (dim > 1 and s2 != 1) or (n > 1 and s1 != dim):
        raise _invalid(f"{name}'s heads must lie side by side in a row (strides {t.stride()})")
    return rows, n, s0 if rows > 1 else n * dim


def _ranges(name: str, t, device: int) -> int:
    torch = _torch()[0]
    _on_device(name, t, device)
    if t.dtype not in (torch.int32, torch.uint32) or t.dim() != 2 or t.shape[1] != 2 or not t.is_contiguous():
        raise _invalid(f"{name} must be a contiguous [sequences, 2] int32 tensor of (start, length)")
    if t.shape[0] > MAX_SEQUENCES:
        raise _invalid(f"{name} names {t.shape[0]} sequences, past 2^30")
    return t.shape[0]


def _stream(stream, device: int):
    """The stream's handle, and the stream itself where it is not the current one."""
    torch, _, raw = _torch()
    if stream is None:
        return raw(device), None
    if hasattr(stream, "cuda_stream"):
        if stream.device.index != device:
            raise _invalid(f"the stream is on {stream.device}, not on cuda:{device}")
        handle, s = stream.cuda_stream, stream
    else:
        handle, s = int(stream), None
    if handle == raw(device):
        return handle, None
    if s is None:
        s = torch.cuda.ExternalStream(handle, device=device) if handle else torch.cuda.default_stream(device)
    return handle, s


def _on(s):
    """A context in which torch allocates on stream `s` (None: already so)."""
    return _HERE if s is None else _torch()[0].cuda.stream(s)


def _in_use(s, *tensors):
    """Keeps the tensors' memory from reuse until what stream `s` has been given has run."""
    if s is not None:
        for t in tensors:
            if t is not None:
                t.record_stream(s)


def _made_on(s, out, device: int):
    """An output allocated on stream `s` for the current one: dropped while work there still reads it, its memory
    is not given out again on `s` before that work has ended."""
    if s is not None:
        out.record_stream(_torch()[0].cuda.current_stream(device))


def _written(out):
    """Tells autograd that a caller's tensor changed: the kernels write through its pointer."""
    _torch()[0].autograd.graph.increment_version(out)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(device: int, dtype: int, heads: int, kv_heads: int, dim: int, scale: float, window: int, ntok: int,
                     prefix: int) -> int:
    s = _lib.GeAttentionShape(dtype, heads, kv_heads, dim, scale, window)
    n = ctypes.c_int64(0)
    _call(_lib.lib().ge_attention_workspace(device, ctypes.byref(s), ntok, prefix, ctypes.byref(n)))
    return n.value


def _attention(q, k, v, prefix_k, prefix_v, q_seqs, kv_seqs, scale, window, out, stream):
    torch = _torch()[0]
    device = _on_device("q", q)
    dtype = q.dtype
    code = _dtype(q)
    if q.dim() != 3:
        raise _invalid(f"q must be [rows, heads, dim], got {list(q.shape)}")
    dim = q.shape[2]
    ntok, heads, q_stride = _heads("q", q, device, dtype, None, dim)
    nkv, kv_heads, k_stride = _heads("k", k, device, dtype, None, dim)
    rows, _, v_stride = _heads("v", v, device, dtype, kv_heads, dim)
    if rows != nkv:
        raise _invalid(f"k has {nkv} rows, v {rows}")
    nseq = _ranges("seqs" if prefix_k is None else "q_seqs", q_seqs, device)
    prefix = pk_stride = pv_stride = 0
    if prefix_k is None:
        if nkv != ntok:
            raise _invalid(f"q has {ntok} rows, k and v {nkv}")
    else:
        prefix, _, pk_stride = _heads("prefix_k", prefix_k, device, dtype, kv_heads, dim)
        rows, _, pv_stride = _heads("prefix_v", prefix_v, device, dtype, kv_heads, dim)
        if rows != prefix:
            raise _invalid(f"prefix_k has {prefix} rows, prefix_v {rows}")
        if _ranges("kv_seqs", kv_seqs, device) != nseq:
            raise _invalid(f"q_seqs names {nseq} sequences, kv_seqs {kv_seqs.shape[0]}")
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    window = min(int(window), MAX_WINDOW)  # no range is longer
    if window < 0:
        raise _invalid("window must not be negative")
    handle, side = _stream(stream, device)
    nbytes = _workspace_bytes(device, code, heads, kv_heads, dim, scale, window, ntok, prefix)
    given = out is not None
    with _on(side):
        if not given:
            out = q.new_empty((ntok, heads, dim))
            out_stride = heads * dim
        else:
            rows, _, out_stride = _heads("out", out, device, dtype, heads, dim)
            if rows != ntok:
                raise _invalid(f"q has {ntok} rows, out {rows}")
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    s = _lib.GeAttentionShape(code, heads, kv_heads, dim, scale, window, q_stride, k_stride, v_stride, pk_stride, pv_stride,
                              out_stride)
    L = _lib.lib()
    if prefix_k is None:
        rc = L.ge_attention_causal(device, s, q.data_ptr(), k.data_ptr(), v.data_ptr(), ntok, q_seqs.data_ptr(), nseq,
                                   out.data_ptr(), ws.data_ptr(), nbytes, handle)
    else:
        rc = L.ge_attention_prefix(device, s, q.data_ptr(), ntok, k.data_ptr(), v.data_ptr(), nkv, prefix_k.data_ptr(),
                                   prefix_v.data_ptr(), prefix, q_seqs.data_ptr(), kv_seqs.data_ptr(), nseq, out.data_ptr(),
                                   ws.data_ptr(), nbytes, handle)
    _call(rc)
    if given:
        _written(out)
    else:
        _made_on(side, out, device)
    _in_use(side, q, k, v, prefix_k, prefix_v, q_seqs, kv_seqs, out)
    return out


def attention_causal(q, k, v, seqs, scale: Optional[float] = None, window: int = 0, out=None, stream=None):
    """Causal attention over packed prompts (ge_attention_causal): row i of a sequence sees the rows
    j <= i of its sequence, with `window` only the last `window` of them (itself included).

    q [T, H, D], k and v [T, KV, D], float16 or bfloat16, D 64, 128 or 256, H a multiple of KV;
    rows may be column ranges of a wider tensor.  `seqs` [n, 2] int32 on the device: (start, length)
    of each sequence, neither negative.  `scale` defaults to 1 / sqrt(D).  Returns `out` [T, H, D], made when
    None (a given one must not overlap the inputs, or is refused);
    rows outside every sequence are left as they were (of a new output: unset)."""
    return _attention(q, k, v, None, None, seqs, seqs, scale, window, out, stream)


def attention_prefix(q, k, v, q_seqs, kv_seqs, prefix_k, prefix_v, scale: Optional[float] = None, out=None, stream=None):
    """Attention of sequences behind one shared prefix (ge_attention_prefix): every query sees all rows
    of prefix_k / prefix_v [P, KV, D] and its own sequence's keys up to its place.

    Sequence s has the query rows q_seqs[s] = (start, n) of q [T, H, D] and the key rows
    kv_seqs[s] = (start, m) of k and v [rows, KV, D]; its queries stand at the end (n = 1 is the step
    of a single token, n = m a whole text).  Rows that see no key give zeros; otherwise as
    attention_causal."""
    if prefix_k is None or prefix_v is None:
        raise _invalid("prefix_k and prefix_v are needed (a prefix may have no rows)")
    return _attention(q, k, v, prefix_k, prefix_v, q_seqs, kv_seqs, scale, 0, out, stream)


@dataclass(frozen=True)
class Q4Weight:
    """A linear layer's 4-bit weights: values [n, k / 2] uint8 (element 2 i in the low half of byte i),
    scales and optionally mins [n, k / group] float16.  w = scale (q - 8), with mins scale q + min."""
    values: Any
    scales: Any
    mins: Any = None

    def __post_init__(self):
        torch = _torch()[0]
        device = _on_device("values", self.values)
        if self.values.dtype != torch.uint8 or self.values.dim() != 2 or not self.values.is_contiguous():
            raise _invalid("values must be a contiguous [n, k / 2] uint8 tensor")
        for name, t in (("scales", self.scales), ("mins", self.mins)):
            if t is None and name == "mins":
                continue
            _on_device(name, t, device)
            if t.dtype != torch.float16 or t.dim() != 2 or t.shape[0] != self.n or not t.is_contiguous():
                raise _invalid(f"{name} must be a contiguous [{self.n}, k / group] float16 tensor")
            _no_gradient(name, t)
        if self.mins is not None and self.mins.shape != self.scales.shape:
            raise _invalid(f"mins must have the shape of scales, {list(self.scales.shape)}")
        groups = self.scales.shape[1]
        if groups == 0 or self.k % groups or self.k // groups not in (32, 64, 128):
            raise _invalid(f"{self.k} weights in {groups} groups: a group must hold 32, 64 or 128")

    @property
    def n(self) -> int:
        return self.values.shape[0]

    @property
    def k(self) -> int:
        return 2 * self.values.shape[1]

    @property
    def group(self) -> int:
        return self.k // self.scales.shape[1]

    @classmethod
    def from_blocks(cls, blocks, kind: str, n: int, k: int, device="cuda") -> "Q4Weight":
        """From n rows of k weights as a GGUF file stores them (`kind` "Q4_0" or "Q4_1"), through
        ge_q4_repack on the host."""
        import torch
        if kind not in Q4_TYPES:
            raise _error(3, f"unsupported tensor type {kind}: Q4_0 and Q4_1 are repacked")
        data = np.frombuffer(blocks, dtype=np.uint8) if isinstance(blocks, (bytes, bytearray, memoryview)) else \
            np.ascontiguousarray(np.asarray(blocks, dtype=np.uint8)).reshape(-1)
        per = 20 if kind == "Q4_1" else 18
        if n < 0 or k <= 0 or k % 32 or data.size != n * (k // 32) * per:
            raise _invalid(f"{n} rows of {k} {kind} weights take {max(n, 0) * (max(k, 0) // 32) * per} bytes, got {data.size}")
        values = np.empty((n, k // 2), np.uint8)
        scales = np.empty((n, k // 32), np.uint16)
        mins = np.empty((n, k // 32), np.uint16) if kind == "Q4_1" else None
        u8, u16 = ctypes.POINTER(ctypes.c_uint8), ctypes.POINTER(ctypes.c_uint16)
        _call(_lib.lib().ge_q4_repack(data.ctypes.data_as(u8), Q4_TYPES[kind], n, k, values.ctypes.data_as(u8),
                                      scales.ctypes.data_as(u16), None if mins is None else mins.ctypes.data_as(u16)))
        half = lambda a: torch.from_numpy(a.view(np.float16)).to(device)
        return cls(torch.from_numpy(values).to(device), half(scales), None if mins is None else half(mins))


def linear_q4(x, weight: Q4Weight, out=None, stream=None):
    """x [rows, k] times the 4-bit weights (ge_linear_q4): out [rows, n] in x's type (float16 or
    bfloat16), for 0 to 64 rows.  x's rows may be a column range of a wider tensor; a given `out` must not
    overlap x or the weights."""
    torch = _torch()[0]
    values, mins = weight.values, weight.mins
    device = _on_device("x", x)
    if values.get_device() != device:
        raise _invalid(f"x is on cuda:{device}, the weight on {values.device}")
    dtype = _dtype(x)
    n, k = values.shape
    k *= 2
    shape = x.shape
    if len(shape) != 2 or shape[1] != k:
        raise _invalid(f"x must be [rows, {k}], got {list(shape)}")
    rows = shape[0]
    if rows > Q4_MAX_ROWS or n > Q4_MAX_N or k > Q4_MAX_K:
        raise _invalid(f"linear_q4 takes up to {Q4_MAX_ROWS} rows, n up to 2^30 and k up to {Q4_MAX_K}; got {rows} rows, n {n}, k {k}")
    x_stride, step = x.stride()
    if step != 1:
        raise _invalid("x's columns must lie side by side")
    _no_gradient("x", x)
    if weight.scales.requires_grad or (mins is not None and mins.requires_grad):  # since the weight was made
        for name, t in (("scales", weight.scales), ("mins", mins)):
            if t is not None:
                _no_gradient(name, t)
    handle, side = _stream(stream, device)
    out_stride = n
    given = out is not None
    if not given:
        with _on(side):
            out = x.new_empty((rows, n))
    else:
        _on_device("out", out, device)
        _no_gradient("out", out)
        if out.dtype != x.dtype or out.shape != (rows, n) or (n > 1 and out.stride(1) != 1):
            raise _invalid(f"out must be a [{rows}, {n}] {x.dtype} tensor with its columns side by side")
        if rows > 1:
            out_stride = out.stride(0)
    _call(_lib.lib().ge_linear_q4(device, dtype, x.data_ptr(), x_stride if rows > 1 else k, rows, k, values.data_ptr(),
                                  weight.scales.data_ptr(), None if mins is None else mins.data_ptr(), weight.group, n,
                                  out.data_ptr(), out_stride, handle))
    if given:
        _written(out)
    else:
        _made_on(side, out, device)
    _in_use(side, x, values, weight.scales, mins, out)
    return out
