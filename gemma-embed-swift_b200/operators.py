"""Operators on torch CUDA tensors, beside the embedding model: attention of causal prompts and of texts
behind a shared prefix, and products of a few rows with 4-bit weights.

They need no model and keep nothing between calls (the entry points are ge_attention_causal,
ge_attention_prefix and ge_linear_q4 of include/gemma_embed.h).  Every call enqueues its work on
`stream` -- a torch stream, a raw cudaStream_t, or None for torch's current stream of the
tensors' device -- and returns without synchronising; it may be captured into a CUDA graph.

    out = attention_causal(q, k, v, seqs)               # q [T, H, D], k and v [T, KV, D]
    last = attention_prefix(q, k, v, q_seqs, kv_seqs, prefix_k, prefix_v)
    y = linear_q4(x, Q4Weight.from_blocks(gguf_bytes, "Q4_0", n, k, device))
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Any, Optional

import numpy as np

from . import _lib

__all__ = ["attention_causal", "attention_prefix", "linear_q4", "Q4Weight"]

Q4_TYPES = {"Q4_0": 2, "Q4_1": 3}  # GGUF tensor type ids (ge_q4_type)


def _error(code: int, message: str):
    from . import GemmaEmbedError
    return GemmaEmbedError(code, message)


def _invalid(message: str):
    return _error(9, f"invalid options: {message}")


def _call(rc: int):
    if rc != 0:
        raise _error(rc, (_lib.lib().ge_last_error(None) or b"").decode())


def _dtype(t) -> int:
    import torch
    if t.dtype == torch.float16:
        return 0
    if t.dtype == torch.bfloat16:
        return 1
    raise _invalid(f"tensors must be float16 or bfloat16, got {t.dtype}")


def _on_device(name: str, t, like=None):
    import torch
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise _invalid(f"{name} must be a CUDA tensor")
    if like is not None and t.device != like.device:
        raise _invalid(f"{name} is on {t.device}, not on {like.device}")


def _heads(name: str, t, like, heads: Optional[int], dim: int) -> int:
    """Checks a [rows, heads, dim] tensor and gives the elements between its rows."""
    _on_device(name, t, like)
    if t.dtype != like.dtype:
        raise _invalid(f"{name} is {t.dtype}, not {like.dtype}")
    if t.dim() != 3 or t.shape[2] != dim or (heads is not None and t.shape[1] != heads):
        want = f"[rows, {heads if heads is not None else 'heads'}, {dim}]"
        raise _invalid(f"{name} must be {want}, got {list(t.shape)}")
    if (dim > 1 and t.stride(2) != 1) or (t.shape[1] > 1 and t.stride(1) != dim):
        raise _invalid(f"{name}'s heads must lie side by side in a row (strides {t.stride()})")
    width = t.shape[1] * dim
    return t.stride(0) if t.shape[0] > 1 else width


def _ranges(name: str, t, like) -> int:
    import torch
    _on_device(name, t, like)
    if t.dtype not in (torch.int32, torch.uint32) or t.dim() != 2 or t.shape[1] != 2 or not t.is_contiguous():
        raise _invalid(f"{name} must be a contiguous [sequences, 2] int32 tensor of (start, length)")
    return t.shape[0]


def _stream(stream, device):
    """The stream's handle, and a torch stream to allocate on."""
    import torch
    if stream is None:
        s = torch.cuda.current_stream(device)
        return s.cuda_stream, s
    if hasattr(stream, "cuda_stream"):
        if stream.device != device:
            raise _invalid(f"the stream is on {stream.device}, not on {device}")
        return stream.cuda_stream, stream
    handle = int(stream)
    if handle == 0:
        return 0, torch.cuda.default_stream(device)
    return handle, torch.cuda.ExternalStream(handle, device=device)


def _attention(q, k, v, prefix_k, prefix_v, q_seqs, kv_seqs, scale, window, out, stream):
    import torch
    _on_device("q", q)
    if q.dim() != 3:
        raise _invalid(f"q must be [rows, heads, dim], got {list(q.shape)}")
    dim = q.shape[2]
    kv_heads = k.shape[1] if hasattr(k, "dim") and k.dim() == 3 else None
    s = _lib.GeAttentionShape()
    s.dtype = _dtype(q)
    s.heads, s.head_dim = q.shape[1], dim
    s.q_stride = _heads("q", q, q, None, dim)
    s.k_stride = _heads("k", k, q, None, dim)
    s.v_stride = _heads("v", v, q, kv_heads, dim)
    s.kv_heads = kv_heads
    if k.shape[0] != v.shape[0]:
        raise _invalid(f"k has {k.shape[0]} rows, v {v.shape[0]}")
    nseq = _ranges("q_seqs" if prefix_k is not None else "seqs", q_seqs, q)
    if prefix_k is None:
        if k.shape[0] != q.shape[0]:
            raise _invalid(f"q has {q.shape[0]} rows, k and v {k.shape[0]}")
    else:
        s.prefix_k_stride = _heads("prefix_k", prefix_k, q, kv_heads, dim)
        s.prefix_v_stride = _heads("prefix_v", prefix_v, q, kv_heads, dim)
        if prefix_k.shape[0] != prefix_v.shape[0]:
            raise _invalid(f"prefix_k has {prefix_k.shape[0]} rows, prefix_v {prefix_v.shape[0]}")
        if _ranges("kv_seqs", kv_seqs, q) != nseq:
            raise _invalid(f"q_seqs names {nseq} sequences, kv_seqs {kv_seqs.shape[0]}")
    s.scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    s.window = int(window)
    device = q.device
    handle, on = _stream(stream, device)
    ntok, prefix = q.shape[0], 0 if prefix_k is None else prefix_k.shape[0]
    L = _lib.lib()
    nbytes = ctypes.c_int64(0)
    with torch.cuda.stream(on):
        if out is None:
            out = torch.empty((ntok, s.heads, dim), dtype=q.dtype, device=device)
        s.out_stride = _heads("out", out, q, s.heads, dim)
        if out.shape[0] != ntok:
            raise _invalid(f"q has {ntok} rows, out {out.shape[0]}")
        _call(L.ge_attention_workspace(device.index, ctypes.byref(s), ntok, prefix, ctypes.byref(nbytes)))
        ws = torch.empty(max(nbytes.value, 1), dtype=torch.uint8, device=device)
        if prefix_k is None:
            _call(L.ge_attention_causal(device.index, ctypes.byref(s), q.data_ptr(), k.data_ptr(), v.data_ptr(), ntok,
                                        q_seqs.data_ptr(), nseq, out.data_ptr(), ws.data_ptr(), nbytes.value, handle))
        else:
            _call(L.ge_attention_prefix(device.index, ctypes.byref(s), q.data_ptr(), ntok, k.data_ptr(), v.data_ptr(),
                                        k.shape[0], prefix_k.data_ptr(), prefix_v.data_ptr(), prefix, q_seqs.data_ptr(),
                                        kv_seqs.data_ptr(), nseq, out.data_ptr(), ws.data_ptr(), nbytes.value, handle))
    return out


def attention_causal(q, k, v, seqs, scale: Optional[float] = None, window: int = 0, out=None, stream=None):
    """Causal attention over packed prompts (ge_attention_causal): row i of a sequence sees the rows
    j <= i of its sequence, with `window` only the last `window` of them (itself included).

    q [T, H, D], k and v [T, KV, D], float16 or bfloat16, D 64, 128 or 256, H a multiple of KV;
    rows may be column ranges of a wider tensor.  `seqs` [n, 2] int32 on the device: (start, length)
    of each sequence.  `scale` defaults to 1 / sqrt(D).  Returns `out` [T, H, D], made when None;
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


@dataclass
class Q4Weight:
    """A linear layer's 4-bit weights: values [n, k / 2] uint8 (element 2 i in the low half of byte i),
    scales and optionally mins [n, k / group] float16.  w = scale (q - 8), with mins scale q + min."""
    values: Any
    scales: Any
    mins: Any = None

    def __post_init__(self):
        import torch
        _on_device("values", self.values)
        if self.values.dtype != torch.uint8 or self.values.dim() != 2 or not self.values.is_contiguous():
            raise _invalid("values must be a contiguous [n, k / 2] uint8 tensor")
        for name, t in (("scales", self.scales), ("mins", self.mins)):
            if t is None and name == "mins":
                continue
            _on_device(name, t, self.values)
            if t.dtype != torch.float16 or t.dim() != 2 or t.shape[0] != self.n or not t.is_contiguous():
                raise _invalid(f"{name} must be a contiguous [{self.n}, k / group] float16 tensor")
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
    bfloat16), for 0 to 64 rows.  x's rows may be a column range of a wider tensor."""
    import torch
    _on_device("x", x, weight.values)
    if x.dim() != 2 or x.shape[1] != weight.k:
        raise _invalid(f"x must be [rows, {weight.k}], got {list(x.shape)}")
    dtype = _dtype(x)
    if x.stride(1) != 1:
        raise _invalid("x's columns must lie side by side")
    rows, n = x.shape[0], weight.n
    handle, on = _stream(stream, x.device)
    with torch.cuda.stream(on):
        if out is None:
            out = torch.empty((rows, n), dtype=x.dtype, device=x.device)
        _on_device("out", out, x)
        if out.dtype != x.dtype or out.shape != (rows, n) or (n > 1 and out.stride(1) != 1):
            raise _invalid(f"out must be a [{rows}, {n}] {x.dtype} tensor with its columns side by side")
        _call(_lib.lib().ge_linear_q4(
            x.device.index, dtype, x.data_ptr(), x.stride(0) if rows > 1 else weight.k, rows, weight.k,
            weight.values.data_ptr(), weight.scales.data_ptr(), None if weight.mins is None else weight.mins.data_ptr(),
            weight.group, n, out.data_ptr(), out.stride(0) if rows > 1 else n, handle))
    return out
