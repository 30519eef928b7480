"""Rope: rotary positions on query and key rows through the C ABI (drkv_rope_*), the rotation of the reference's
rope_kernel (src/machina/layer_attention.cu:32-79) for rows in the caller's tensors."""
from __future__ import annotations

import ctypes as C
from typing import Optional

import numpy as np

from . import capi
from .capi import RopeConfig, RopeRows, check
from .engine import _stream

LAYOUTS = {"halves": 0, "pairs": 1}
SCALINGS = {"none": 0, "linear": 1, "base": 2, "bands": 3, "ramp": 4}
DTYPES = {"f16": capi.F16, "fp16": capi.F16, "bf16": capi.BF16}


class Rope:
    """One rotation: its frequencies live on the device, `apply` runs it.  See drkv_rope_config for the parameters."""

    def __init__(self, *, head_dim: int, rotary_dim: Optional[int] = None, theta: float = 10000.0, layout: str = "halves",
                 dtype: str = "bf16", scaling: str = "none", factor: float = 1.0, original_context: int = 0,
                 low_freq_factor: float = 1.0, high_freq_factor: float = 4.0, beta_fast: float = 32.0,
                 beta_slow: float = 1.0, attention_factor: float = 0.0, device: int = 0):
        self.h = None
        for name, table, value in (("layout", LAYOUTS, layout), ("scaling", SCALINGS, scaling), ("dtype", DTYPES, dtype)):
            if value not in table:
                raise ValueError(f"{name} must be one of {sorted(table)}, not {value!r}")
        self.lib = capi.load_library()
        self.head_dim, self.device, self.dtype = head_dim, device, DTYPES[dtype]
        cfg = RopeConfig(head_dim, head_dim if rotary_dim is None else rotary_dim, LAYOUTS[layout], self.dtype,
                         SCALINGS[scaling], device, original_context, low_freq_factor, high_freq_factor, beta_fast,
                         beta_slow, attention_factor, theta, factor)
        h = C.c_void_p()
        check(self.lib.drkv_rope_create(C.byref(cfg), C.byref(h)))
        self.h = h

    def close(self):
        if getattr(self, "h", None):
            self.lib.drkv_rope_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def frequencies(self) -> np.ndarray:
        """Radians per position of every pair."""
        n = check(self.lib.drkv_rope_frequencies(self.h, None, 0))
        out = np.empty(n, dtype=np.float64)
        check(self.lib.drkv_rope_frequencies(self.h, out.ctypes.data_as(C.POINTER(C.c_double)), n))
        return out

    def _rows(self, src, dst, n_tokens, name) -> RopeRows:
        shape, strides, to_shape, to_strides = src.shape, src.stride(), dst.shape, dst.stride()
        if (len(shape) != 3 or shape[0] != n_tokens or shape[2] != self.head_dim or to_shape != shape or
                src.dtype is not self._torch_dtype or dst.dtype is not self._torch_dtype or strides[2] != 1 or to_strides[2] != 1 or
                src.get_device() != self.device or dst.get_device() != self.device):
            raise ValueError(f"{name} and out_{name} must be tensors [{n_tokens}, heads, {self.head_dim}] of {self._torch_dtype} on "
                             f"cuda:{self.device} with a contiguous last dimension, not {tuple(shape)} {src.dtype} {src.device} and "
                             f"{tuple(to_shape)} {dst.dtype} {dst.device}")
        return RopeRows(src.data_ptr(), dst.data_ptr(), shape[1], strides[0], strides[1], to_strides[0], to_strides[1])

    def _new(self, like, stream):
        import torch
        if stream is None:
            return torch.empty(like.shape, dtype=like.dtype, device=like.device)
        # the allocator may hand out memory that earlier work of the stream it believes to be current still uses
        with torch.cuda.stream(torch.cuda.ExternalStream(_stream(stream), device=self.device)):
            return torch.empty(like.shape, dtype=like.dtype, device=like.device)

    def apply(self, pos, q=None, k=None, *, out_q=None, out_k=None, inverse: bool = False, stream=None):
        """Rotates q and k, tensors [n_tokens, heads, head_dim] of any token and head strides, by the int32 positions
        `pos` [n_tokens]; into out_q / out_k (new contiguous tensors by default; the input itself for in place).
        inverse=True applies the transpose, the gradient; apply itself is not recorded for autograd, tensors that require one
        are refused while gradients are enabled.  Runs on `stream`, by default the device's current one; new outputs
        belong to it.  Returns (out_q, out_k)."""
        import torch
        if q is None and k is None:
            raise ValueError("nothing to rotate: give q, k or both")
        if (q is None and out_q is not None) or (k is None and out_k is not None):
            raise ValueError("an output without its input")
        if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, out_q, out_k)):
            raise ValueError("apply is not recorded for autograd and would drop the gradient: call it under torch.no_grad(); "
                             "the gradient of its inputs is apply(..., inverse=True) of the outputs'")
        if pos.dtype is not torch.int32 or pos.dim() != 1 or not pos.is_contiguous() or pos.get_device() != self.device:
            raise ValueError(f"pos must be a contiguous int32 vector on cuda:{self.device}")
        self._torch_dtype = torch.float16 if self.dtype == capi.F16 else torch.bfloat16
        n = pos.shape[0]
        q_rows = k_rows = None
        if q is not None:
            if out_q is None:
                out_q = self._new(q, stream)
            q_rows = C.byref(self._rows(q, out_q, n, "q"))
        if k is not None:
            if out_k is None:
                out_k = self._new(k, stream)
            k_rows = C.byref(self._rows(k, out_k, n, "k"))
        check(self.lib.drkv_rope_apply(self.h, n, pos.data_ptr(), q_rows, k_rows, 1 if inverse else 0,
                                       _stream(torch.cuda.current_stream(self.device) if stream is None else stream)))
        return out_q, out_k
