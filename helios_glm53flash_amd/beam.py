"""One step of beam search over libhx_exl3.so: selection over beams and vocabulary from the head's logits, and the
surviving beams' states copied from their parents.

    w4.embed / gather_rows -> layers -> lm_head (exl3.gemm or w4.gemm) -> select -> (the caller keeps the finished ones) -> reorder
"""
from __future__ import annotations

import ctypes as C
from functools import lru_cache
from typing import Optional

import torch

from ._lib import check, lib
from .exl3 import _need, _ptr, _stream
from .w4 import _on_one_device, call_workspace

_DTYPES = {torch.float16: 0, torch.float32: 1}


@lru_cache(maxsize=4096)
def _select_workspace_bytes(batch: int, beams: int, vocab: int, n: int) -> int:
    return lib.hx_beam_select_workspace_size(batch, beams, vocab, n)


def select(logits: torch.Tensor, cum: torch.Tensor, done: Optional[torch.Tensor], scores: torch.Tensor,
           parents: torch.Tensor, tokens: torch.Tensor, batch: int, beams: int, vocab: int, n: int, eos: int = 0,
           stream=None) -> None:
    """The n best continuations of each sequence: score = cum + log_softmax(logits), descending, the lowest
    beam * vocab + token first among equals, off by 4e-6 + 3e-7 p at most beside the rounding to fp32 (p pieces of 4096 logits a
    workgroup, 1 up to 27 rows of 151552), into scores (fp32), parents (beam within the sequence) and tokens (int64),
    each [batch][n].  logits [batch * beams][>= vocab] fp16 or fp32, rows at any stride >= vocab; cum fp32 [batch * beams]; done
    (uint8 or bool, optional) marks finished beams, which go on with eos at an unchanged score.  Forbidden tokens have logit
    -inf, dead beams cum -inf; places that no candidate fills get -inf, -1, -1.  scores may be cum itself where n == beams."""
    if not isinstance(logits, torch.Tensor) or logits.dtype not in _DTYPES or not logits.is_cuda or logits.dim() != 2:
        raise ValueError("select: logits must be a 2-d float16 or float32 device tensor")
    if max(batch, beams, vocab, n) >> 31 or done is not None and eos >> 31 not in (0, -1):
        raise ValueError("select: batch, beams, vocab, n and eos must fit 32 bits")
    rows = batch * beams
    height, width = logits.shape
    if batch < 0 or beams < 1 or vocab < 1 or n < 1 or height < rows or width < vocab:
        raise ValueError("select: logits smaller than [batch * beams][vocab]")
    ld, step = logits.stride()
    if height < 2:
        ld = max(vocab, ld)
    if vocab > 1 and step != 1 or ld < vocab:
        raise ValueError("select: the logits of a row must be consecutive and rows must not overlap")
    _need(cum, "cum", (torch.float32,))
    _need(scores, "scores", (torch.float32,))
    _need(parents, "parents", (torch.int64,))
    _need(tokens, "tokens", (torch.int64,))
    if done is not None:
        _need(done, "done", (torch.uint8, torch.bool))
        if done.numel() < rows:
            raise ValueError("select: done smaller than batch * beams")
    places = batch * n
    if cum.numel() < rows or scores.numel() < places or parents.numel() < places or tokens.numel() < places:
        raise ValueError("select: cum / outputs smaller than batch * beams / batch * n")
    _on_one_device(logits, cum, done, scores, parents, tokens)
    st = _stream(stream)
    ws = call_workspace(_select_workspace_bytes(batch, beams, vocab, n), logits.device, st)
    check(lib.hx_beam_select(logits.data_ptr(), cum.data_ptr(), _ptr(done), scores.data_ptr(), parents.data_ptr(),
                             tokens.data_ptr(), batch, beams, vocab, n, ld, eos, _DTYPES[logits.dtype], st, ws.data_ptr(),
                             ws.numel()), "hx_beam_select")


def _merge(dims, run):
    """Dimensions (count, src stride, dst stride) in bytes, outermost first, merged where both sides allow it: (merged
    dimensions, bytes of the consecutive run inside them), starting from a run of `run` bytes (None: no run, the dimensions
    outside the beams')."""
    merged = []  # innermost first
    for n, s, d in reversed(dims):
        if n == 1:
            continue
        if run is not None and not merged and s == d == run:
            run *= n
        elif merged and (s, d) == (merged[-1][0] * merged[-1][1], merged[-1][0] * merged[-1][2]):
            merged[-1] = (merged[-1][0] * n, *merged[-1][1:])
        else:
            merged.append((n, s, d))
    if len(merged) > 1:
        raise ValueError("reorder: the dimensions on one side of dim do not reduce to a single stride in src and dst")
    return (merged[0] if merged else (1, 0, 0)), run


@lru_cache(maxsize=1024)
def _geometry(src_shape, src_stride, dst_shape, dst_stride, e, dim, rows, out_rows):
    """(outer, inner, bytes, source strides, destination strides) for the C call."""
    want = list(src_shape)
    want[dim] = out_rows
    if src_shape[dim] != rows or list(dst_shape) != want:
        raise ValueError("reorder: src must have batch * beams rows along dim, dst batch * out_beams and src's other extents")
    if 0 in want:
        return None
    dims = [(n, s * e, d * e) for n, s, d in zip(src_shape, src_stride, dst_stride)]
    (inner, si, di), run = _merge(dims[dim + 1:], e)
    (outer, so, do), _ = _merge(dims[:dim], None)
    three = C.c_int64 * 3
    return outer, inner, run, three(so, dims[dim][1], si), three(do, dims[dim][2], di)


def reorder(src: torch.Tensor, parents: torch.Tensor, dst: torch.Tensor, batch: int, beams: int, out_beams: int,
            dim: int = 0, stream=None) -> None:
    """dst[.., b * out_beams + j, ..] = src[.., b * beams + parents[b][j], ..] along dimension dim, for states of any real type
    and shape: dim counts batch * beams rows in src and batch * out_beams in dst, the other dimensions agree.  Views are
    accepted (a cache filled below its capacity) as long as the dimensions on either side of dim reduce to one stride each.
    Rows whose parent lies outside [0, beams) are left as they were; src and dst may not overlap."""
    for t, name in ((src, "src"), (dst, "dst")):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError(f"reorder: {name} must be a device tensor")
    _need(parents, "parents", (torch.int64,))
    if src.dtype != dst.dtype or src.is_complex() or src.dim() != dst.dim() or not -src.dim() <= dim < src.dim():
        raise ValueError("reorder: src and dst must have the same (real) type and dimensions, dim among them")
    if max(batch, beams, out_beams) >> 31:
        raise ValueError("reorder: batch, beams and out_beams must fit 32 bits")
    if batch < 0 or beams < 1 or out_beams < 0 or parents.numel() < batch * out_beams:
        raise ValueError("reorder: parents smaller than batch * out_beams")
    _on_one_device(src, parents, dst)
    g = _geometry(src.shape, src.stride(), dst.shape, dst.stride(), src.element_size(), dim % src.dim(), batch * beams,
                  batch * out_beams)
    if g is None:
        return
    outer, inner, run, ss, ds = g
    check(lib.hx_beam_reorder(src.data_ptr(), parents.data_ptr(), dst.data_ptr(), batch, beams, out_beams, outer, inner, run,
                              ss, ds, _stream(stream)), "hx_beam_reorder")


__all__ = ["select", "reorder"]
