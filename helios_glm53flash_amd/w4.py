"""Linears over plain 4-bit codes with group scales (libhx_exl3.so): the counterpart of exl3.gemm for projections and heads
that are not trellis coded, and the lookup of single rows (a head that is the embedding too).

    W[n][k] = scales[n][k // group] * (q[n][k] - zeros[n][k // group])      zeros 8 where there are none

`pack` lays codes out once, when a layer is loaded.  Buffers are torch tensors on the current HIP device.
"""
from __future__ import annotations

import ctypes as C
from contextlib import nullcontext
from dataclasses import dataclass
from functools import lru_cache
from typing import Optional

import torch

from ._lib import W4WordsC, check, lib
from .exl3 import _GEMM_EXTRA, _get_device, _need, _ptr, _stream, _workspaces, workspace

_is_capturing = torch._C._cuda_isCurrentStreamCapturing
COUNTER_BYTES = 64 * 1024  # arrival counters at the start of a workspace
_NIBBLE_K = (0, 2, 4, 6, 1, 3, 5, 7)  # the k of an octet that each nibble of its word holds, lowest nibble first


def pack(q: torch.Tensor) -> torch.Tensor:
    """int32 words [N][16 * ceil(K / 128)] of codes q uint8 [N][K] (0..15), K a multiple of 32."""
    if q.dim() != 2 or q.dtype != torch.uint8:
        raise ValueError("pack: q must be uint8 [N][K]")
    N, K = q.shape
    if K == 0 or K % 32:
        raise ValueError("pack: K must be a positive multiple of 32")
    if q.numel() and int(q.max()) > 15:
        raise ValueError("pack: codes must be in 0..15")
    q = torch.nn.functional.pad(q, (0, -K % 128))
    octets = q.view(N, q.shape[1] // 128, 4, 4, 8).transpose(2, 3)  # octet 4 j + g of a block is word 4 g + j
    words = torch.zeros(octets.shape[:-1], dtype=torch.int32, device=q.device)
    for i, k in enumerate(_NIBBLE_K):
        words |= octets[..., k].to(torch.int32) << (4 * i)
    return words.reshape(N, q.shape[1] // 8).contiguous()


def unpack(words: torch.Tensor, K: int) -> torch.Tensor:
    """The codes uint8 [N][K] of int32 words: the inverse of pack."""
    if words.dim() != 2 or words.dtype != torch.int32 or K <= 0 or K % 32 or words.shape[1] != (K + 127) // 128 * 16:
        raise ValueError("unpack: words must be int32 [N][16 * ceil(K / 128)], K a positive multiple of 32")
    w = words.view(words.shape[0], words.shape[1] // 16, 4, 4).transpose(2, 3)
    q = torch.empty((*w.shape, 8), dtype=torch.uint8, device=words.device)
    for i, k in enumerate(_NIBBLE_K):
        q[..., k] = ((w >> (4 * i)) & 15).to(torch.uint8)
    return q.reshape(words.shape[0], words.shape[1] * 8)[:, :K].contiguous()


@dataclass(frozen=True)
class W4Words:
    """One linear: words int32 [N][16 * ceil(K / 128)] (see pack), scales fp16 [N][ceil(K / group)], zeros uint8 of that
    shape or None (8), the number K of input features, the group size (a power of two >= 32).  The tensors are checked and
    the C descriptor is made once, here: that took 1.6 of the 7 us that a small call costs on the host."""
    words: torch.Tensor
    scales: torch.Tensor
    zeros: Optional[torch.Tensor]
    in_features: int
    group: int

    def __post_init__(self):
        z, K, group = self.zeros, self.in_features, self.group
        if K <= 0 or K % 32 or group < 32 or group & (group - 1):
            raise ValueError("W4Words: K must be a positive multiple of 32 and group a power of two of at least 32")
        _need(self.words, "words", (torch.int32,))
        _need(self.scales, "scales", (torch.float16,))
        if self.words.dim() != 2 or self.words.shape[1] != (K + 127) // 128 * 16:
            raise ValueError("W4Words: words must be [N][16 * ceil(K / 128)]")
        shape = (self.words.shape[0], (K + group - 1) // group)
        if self.scales.shape != shape:
            raise ValueError(f"W4Words: scales must be {shape}")
        if z is not None:
            _need(z, "zeros", (torch.uint8,))
            if z.shape != shape:
                raise ValueError(f"W4Words: zeros must be {shape}")
        if len({t.get_device() for t in (self.words, self.scales, z) if t is not None}) != 1:
            raise ValueError("W4Words: words, scales and zeros must be on one device")
        ptrs = (self.words.data_ptr(), self.scales.data_ptr(), _ptr(z))
        object.__setattr__(self, "_ptrs", ptrs)
        object.__setattr__(self, "_c", W4WordsC(*ptrs, group))
        object.__setattr__(self, "device_index", self.words.get_device())
        object.__setattr__(self, "out_features", shape[0])

    def c(self) -> W4WordsC:
        """The C descriptor (made again if a tensor was given other memory)."""
        if (self.words.data_ptr(), self.scales.data_ptr(), _ptr(self.zeros)) != self._ptrs:
            self.__post_init__()
        return self._c


def _on_one_device(*tensors) -> None:
    dev = _get_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"tensors must be on the current device (cuda:{dev}), got {t.device}")


def _weights_here(w: W4Words) -> None:
    if w.device_index != _get_device():
        raise ValueError(f"the weights are on cuda:{w.device_index}, the current device is cuda:{_get_device()}")


@lru_cache(maxsize=4096)
def _gemm_workspace_bytes(M: int, N: int, K: int) -> int:
    return lib.hx_w4_gemm_workspace_size(M, N, K)


# (device, stream) -> (capture, workspace) of the last capture there.  Held so that a capture's calls share it and its counters are
# cleared once (2 us a call otherwise).
_captured: dict[tuple, tuple] = {}


def call_workspace(nbytes: int, device: torch.device, st: int) -> torch.Tensor:
    """A call's workspace on stream st: the stream's own one, or, where st is being captured, memory of the graph's whose
    counters each replay clears ahead of the first call, so that the graph depends on no buffer that a later call may replace."""
    here = st == _stream(None)
    if not here or _is_capturing():
        capture, key = lib.hx_capture_id(st), (_get_device(), st)
        if capture:
            held = _captured.get(key)
            if held is None or held[0] != capture or held[1].numel() < nbytes:
                with nullcontext() if here else torch.cuda.stream(torch.cuda.ExternalStream(st, device=device)):
                    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
                    ws[:COUNTER_BYTES].zero_()
                _captured[key] = held = (capture, ws)
            return held[1]
    ws = _workspaces.get((_get_device(), st))
    if ws is not None and ws.numel() >= nbytes:
        return ws
    # the bytes behind every workspace, which hold a linear's splits, are enough here too
    return workspace(max(0, nbytes - _GEMM_EXTRA), device, st)


def gemm(y: torch.Tensor, x: torch.Tensor, w: W4Words, M: int, N: int, K: int, y_fp32: bool = False, stream=None) -> None:
    """y[m][n] = sum_k x[m][k] W[n][k]: x fp16 [M][K], y fp32 or fp16 [M][N], any M (M = 0 is a no-op); y may not
    overlap x.  Shapes that split K over workgroups do so in the stream's workspace (exl3.workspace, which never grows for it)."""
    _need(x, "x", (torch.float16,))
    _need(y, "y", (torch.float32,) if y_fp32 else (torch.float16,))
    if M >> 31:
        raise ValueError("gemm: M must be non-negative and fit 32 bits")
    if x.numel() < M * K or y.numel() < M * N:
        raise ValueError("x / y smaller than M*K / M*N")
    if w.in_features != K or w.out_features != N:
        raise ValueError("W4Words shapes do not match K, N")
    _on_one_device(x, y)
    _weights_here(w)
    st = _stream(stream)
    need = _gemm_workspace_bytes(M, N, K)
    ws = call_workspace(need, x.device, st) if need else None
    check(lib.hx_w4_gemm(y.data_ptr(), x.data_ptr(), C.byref(w.c()), M, N, K, int(y_fp32), st, _ptr(ws),
                         ws.numel() if ws is not None else 0), "hx_w4_gemm")


def embed(w: W4Words, tokens: torch.Tensor, out: torch.Tensor, n: int, scale: float = 1.0, stream=None) -> None:
    """out[t] = scale * W[tokens[t]] for t < n (tokens int64; out fp16 or fp32 rows of K); zeros for a token outside
    [0, N)."""
    _need(tokens, "tokens", (torch.int64,))
    _need(out, "out", (torch.float16, torch.float32))
    if n >> 31:
        raise ValueError("embed: n must be non-negative and fit 32 bits")
    if tokens.numel() < n or out.numel() < n * w.in_features:
        raise ValueError("embed: tokens / out smaller than n / n*K")
    _on_one_device(tokens, out)
    _weights_here(w)
    check(lib.hx_w4_embed(C.byref(w.c()), tokens.data_ptr(), out.data_ptr(), n, w.out_features, w.in_features, scale,
                          int(out.dtype == torch.float32), _stream(stream)), "hx_w4_embed")


__all__ = ["W4Words", "pack", "unpack", "gemm", "embed"]
