"""Rope: rotary positions on query and key rows through the C ABI (drkv_rope_*), the rotation of the reference's
rope_kernel (src/machina/layer_attention.cu:32-79) for rows in the caller's tensors."""
from __future__ import annotations

import ctypes as C
from typing import Optional

import numpy as np

from . import capi
from .capi import RopeConfig, RopeRows, check
from .engine import _ptr, _stream

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
        import torch
        want = torch.float16 if self.dtype == capi.F16 else torch.bfloat16
        for what, t in ((name, src), (f"out_{name}", dst)):
            if t.dim() != 3 or t.shape[0] != n_tokens or t.shape[2] != self.head_dim:
                raise ValueError(f"{what} must have shape [{n_tokens}, heads, {self.head_dim}], not {tuple(t.shape)}")
            if t.dtype != want:
                raise ValueError(f"{what} must be {want}, not {t.dtype}")
            if t.device.type != "cuda" or t.device.index != self.device:
                raise ValueError(f"{what} must be on cuda:{self.device}, not {t.device}")
            if t.stride(2) != 1:
                raise ValueError(f"the last dimension of {what} must be contiguous")
        if dst.shape != src.shape:
            raise ValueError(f"out_{name} must have the shape of {name}")
        return RopeRows(_ptr(src), _ptr(dst), src.shape[1], src.stride(0), src.stride(1), dst.stride(0), dst.stride(1))

    def apply(self, pos, q=None, k=None, *, out_q=None, out_k=None, inverse: bool = False, stream=None):
        """Rotates q and k, tensors [n_tokens, heads, head_dim] of any token and head strides, by the int32 positions
        `pos` [n_tokens]; into out_q / out_k (new contiguous tensors by default; the input itself for in place).
        inverse=True applies the transpose, the gradient.  Returns (out_q, out_k)."""
        import torch
        if q is None and k is None:
            raise ValueError("nothing to rotate: give q, k or both")
        if pos.dtype != torch.int32 or pos.dim() != 1 or not pos.is_contiguous() or pos.device.index != self.device:
            raise ValueError(f"pos must be a contiguous int32 vector on cuda:{self.device}")
        rows = []
        outs = []
        for name, src, dst in (("q", q, out_q), ("k", k, out_k)):
            if src is None:
                if dst is not None:
                    raise ValueError(f"out_{name} without {name}")
                rows.append(None)
                outs.append(None)
                continue
            if dst is None:
                dst = torch.empty(src.shape, dtype=src.dtype, device=src.device)
            rows.append(self._rows(src, dst, pos.shape[0], name))
            outs.append(dst)
        ref = [None if r is None else C.byref(r) for r in rows]
        check(self.lib.drkv_rope_apply(self.h, pos.shape[0], _ptr(pos), ref[0], ref[1], 1 if inverse else 0, _stream(stream)))
        return outs[0], outs[1]
