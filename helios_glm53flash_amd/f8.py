"""Linears in 8-bit floating point (e4m3) with a scale for each block of 128, and what feeds them (libhx_exl3.so): the counterpart of
exl3.gemm and w4.gemm for a model whose projections and dense layers are stored that way.

    rms_norm -> gemm (projections) -> attention -> quantize -> gemm -> rms_norm -> gate_up -> gemm (down)

Input rows have a scale for each 128 consecutive k, weights one for each 128 x 128; the last blocks may be short.
    a = max(largest |v| of the block, 2^-100)      scale = a / 448      code = e4m3(v * (448 / a)), to nearest even
A block with a NaN or an infinity stands for NaN throughout.  K is a multiple of 16.  Buffers are torch tensors on the current HIP device.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from functools import lru_cache
from typing import Optional

import torch

from ._lib import F8BlocksC, check, lib
from .exl3 import _get_device, _need, _ptr, _stream
from .w4 import _on_one_device, call_workspace

BLOCK = 128
F8 = torch.float8_e4m3fn
_DTYPES = {torch.float16: 0, torch.float32: 1}


@dataclass(frozen=True)
class F8Blocks:
    """One linear: codes float8_e4m3fn [N][K], scales fp32 [ceil(N / 128)][ceil(K / 128)].  The tensors are checked and the C
    descriptor is made once, here."""
    codes: torch.Tensor
    scales: torch.Tensor

    def __post_init__(self):
        _need(self.codes, "codes", (F8,))
        _need(self.scales, "scales", (torch.float32,))
        if self.codes.dim() != 2 or self.codes.shape[0] < 1 or self.codes.shape[1] < 1 or self.codes.shape[1] % 16:
            raise ValueError("F8Blocks: codes must be [N][K], K a positive multiple of 16")
        N, K = self.codes.shape
        shape = ((N + BLOCK - 1) // BLOCK, (K + BLOCK - 1) // BLOCK)
        if self.scales.shape != shape:
            raise ValueError(f"F8Blocks: scales must be {shape}")
        if self.codes.get_device() != self.scales.get_device():
            raise ValueError("F8Blocks: codes and scales must be on one device")
        ptrs = (self.codes.data_ptr(), self.scales.data_ptr())
        object.__setattr__(self, "_ptrs", ptrs)
        object.__setattr__(self, "_c", F8BlocksC(*ptrs))
        object.__setattr__(self, "device_index", self.codes.get_device())
        object.__setattr__(self, "out_features", N)
        object.__setattr__(self, "in_features", K)

    def c(self) -> F8BlocksC:
        """The C descriptor (made again if a tensor was given other memory)."""
        if (self.codes.data_ptr(), self.scales.data_ptr()) != self._ptrs:
            self.__post_init__()
        return self._c


def _blocks_here(w: F8Blocks, N: int, K: int) -> None:
    if w.out_features != N or w.in_features != K:
        raise ValueError("F8Blocks shapes do not match K, N")
    if w.device_index != _get_device():
        raise ValueError(f"the weights are on cuda:{w.device_index}, the current device is cuda:{_get_device()}")


def _extents(who: str, M: int, K: int) -> int:
    """Blocks of a row."""
    if M >> 31 or K < 1 or K >> 31:
        raise ValueError(f"{who}: M must be non-negative, K positive, and both must fit 32 bits")
    return (K + BLOCK - 1) // BLOCK


def _rows(who: str, x: torch.Tensor, M: int, K: int) -> int:
    """Elements from one row of x [>= M][K] to the next."""
    if not isinstance(x, torch.Tensor) or x.dtype not in _DTYPES or not x.is_cuda or x.dim() != 2:
        raise ValueError(f"{who}: x must be a 2-d float16 or float32 device tensor")
    height, width = x.shape
    ld, step = x.stride()
    if height < M or width < K:
        raise ValueError(f"{who}: x smaller than [M][K]")
    if height < 2:
        ld = (max(ld, K) + 7) // 8 * 8  # of one row, which has no next
    if K > 1 and step != 1 or ld < K:
        raise ValueError(f"{who}: the values of a row of x must be consecutive and rows must not overlap")
    return ld


def _codes(who: str, q: torch.Tensor, scales: torch.Tensor, M: int, K: int, kb: int, name: str = "q", scales_name: str = "scales") -> None:
    _need(q, name, (F8,))
    _need(scales, scales_name, (torch.float32,))
    if q.numel() < M * K or scales.numel() < M * kb:
        raise ValueError(f"{who}: codes / scales smaller than M * K / M * ceil(K / 128): {name}, {scales_name}")


def quantize(x: torch.Tensor, q: torch.Tensor, scales: torch.Tensor, M: int, K: int, stream=None) -> None:
    """q (float8_e4m3fn [M][K]) and scales (fp32 [M][ceil(K / 128)]) of x, fp16 or fp32 [M][K] with rows at any stride that is a
    multiple of 8."""
    kb = _extents("quantize", M, K)
    ld = _rows("quantize", x, M, K)
    _codes("quantize", q, scales, M, K, kb)
    _on_one_device(x, q, scales)
    check(lib.hx_f8_quantize(x.data_ptr(), q.data_ptr(), scales.data_ptr(), M, K, ld, _DTYPES[x.dtype], _stream(stream)), "hx_f8_quantize")


def rms_norm(x: torch.Tensor, weight: torch.Tensor, M: int, K: int, eps: float, residual: Optional[torch.Tensor] = None,
             out: Optional[torch.Tensor] = None, y: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None,
             scales: Optional[torch.Tensor] = None, stream=None) -> None:
    """h = x + residual, rounded to residual's type, into out (residual itself: in place); n = h / sqrt(mean(h^2) + eps) * weight;
    y (fp16) = n; q and scales: blocks of n before that rounding.  x as in quantize; residual and out fp16 or fp32 [M][K], or neither
    (h = x); weight fp16 or fp32 [K]; y, or q and scales, or all three.  Rows of zeros give zeros, but NaN where eps is 0."""
    kb = _extents("rms_norm", M, K)
    ld = _rows("rms_norm", x, M, K)
    _need(weight, "weight", (torch.float16, torch.float32))
    if weight.numel() != K:
        raise ValueError("rms_norm: weight must have K values")
    if (residual is None) != (out is None) or (q is None) != (scales is None):
        raise ValueError("rms_norm: residual and out, and q and scales, are given together")
    if residual is not None:
        _need(residual, "residual", (torch.float16, torch.float32))
        _need(out, "out", (residual.dtype,))
        if residual.numel() < M * K or out.numel() < M * K:
            raise ValueError("rms_norm: residual / out smaller than M * K")
    if y is not None:
        _need(y, "y", (torch.float16,))
        if y.numel() < M * K:
            raise ValueError("rms_norm: y smaller than M * K")
    if q is not None:
        _codes("rms_norm", q, scales, M, K, kb)
    _on_one_device(x, weight, residual, out, y, q, scales)
    check(lib.hx_f8_rms_norm(x.data_ptr(), ld, _DTYPES[x.dtype], _ptr(residual), _ptr(out),
                             0 if residual is None else _DTYPES[residual.dtype], weight.data_ptr(), _DTYPES[weight.dtype], _ptr(y),
                             _ptr(q), _ptr(scales), M, K, eps, _stream(stream)), "hx_f8_rms_norm")


@lru_cache(maxsize=4096)
def _gemm_workspace_bytes(M: int, N: int, K: int) -> int:
    return lib.hx_f8_gemm_workspace_size(M, N, K)


@lru_cache(maxsize=4096)
def _gate_up_workspace_bytes(M: int, N: int, K: int) -> int:
    return lib.hx_f8_gate_up_workspace_size(M, N, K)


def gemm(y: torch.Tensor, x: torch.Tensor, x_scales: torch.Tensor, w: F8Blocks, M: int, N: int, K: int, y_fp32: bool = False,
         stream=None, exact: bool = False) -> None:
    """y[m][n] = sum_k x[m][k] W[n][k] over the values that the codes and scales stand for: x and x_scales as quantize gives them,
    y fp32 or fp16 [M][N], any M (M = 0 is a no-op).  fp32 outputs, and up to 8 rows, come from exact products; fp16 outputs of more rows cut those
    of 8 consecutive k at 2^-13 of their largest (some 2^-16 of the outputs' size), but where `exact` asks for the others' way.  Shapes that split K over workgroups do so in the stream's workspace."""
    kb = _extents("gemm", M, K)
    _codes("gemm", x, x_scales, M, K, kb, "x", "x_scales")
    _need(y, "y", (torch.float32,) if y_fp32 else (torch.float16,))
    if y.numel() < M * N:
        raise ValueError("gemm: y smaller than M * N")
    _blocks_here(w, N, K)
    _on_one_device(x, x_scales, y)
    st = _stream(stream)
    need = _gemm_workspace_bytes(M, N, K)
    ws = call_workspace(need, x.device, st) if need else None
    entry, name = (lib.hx_f8_gemm_exact, "hx_f8_gemm_exact") if exact else (lib.hx_f8_gemm, "hx_f8_gemm")
    check(entry(y.data_ptr(), x.data_ptr(), x_scales.data_ptr(), C.byref(w.c()), M, N, K, int(y_fp32), st, _ptr(ws),
                ws.numel() if ws is not None else 0), name)


def gate_up(q: torch.Tensor, scales: torch.Tensor, x: torch.Tensor, x_scales: torch.Tensor, gate: F8Blocks, up: F8Blocks, M: int,
            N: int, K: int, limit: float = 10.0, stream=None) -> None:
    """The first half of a gated feed-forward block: g = x gate^T, u = x up^T, v = silu(min(g, limit)) * clamp(u, -limit, limit), and q
    (float8_e4m3fn [M][N]), scales (fp32 [M][ceil(N / 128)]) the blocks of v, ready for gemm with the down projection.  N is a multiple of
    16; limit = inf does not clamp."""
    kb = _extents("gate_up", M, K)
    nb = _extents("gate_up", M, N)
    _codes("gate_up", x, x_scales, M, K, kb, "x", "x_scales")
    _codes("gate_up", q, scales, M, N, nb)
    _blocks_here(gate, N, K)
    _blocks_here(up, N, K)
    _on_one_device(x, x_scales, q, scales)
    st = _stream(stream)
    need = _gate_up_workspace_bytes(M, N, K)
    ws = call_workspace(need, x.device, st) if need else None
    check(lib.hx_f8_gate_up(q.data_ptr(), scales.data_ptr(), x.data_ptr(), x_scales.data_ptr(), C.byref(gate.c()), C.byref(up.c()), M,
                            N, K, limit, st, _ptr(ws), ws.numel() if ws is not None else 0), "hx_f8_gate_up")


__all__ = ["F8Blocks", "quantize", "rms_norm", "gemm", "gate_up"]
