"""Token operators on the layer's feature maps, backed by libdcnv2.so: what a transformer that
reads the maps (a detection decoder, a language model with image tokens) does with them.

dcnv2_qk_norm_rotary   RMS norm of each query and key head and its rotation by the token's position
                       on one to four axes (text; row and column; frame or level, row, column)
dcnv2_cross_attention  attention of queries to the states of another sequence: many queries or
                       single tokens, grouped heads, lengths and masks of padded images
rotary_axes            frequency table and axis of each rotated pair, made once per model
level_positions        (level, row, column) of every pixel of a pyramid's levels

Both operators take strided torch CUDA tensors (views of one projection, caches laid out heads
first), run on the current torch stream of the tensors' device unless a stream is given, and raise
DCNv2Error on any failure. They are inference operators, as the layer is: no gradients.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import math
from typing import Sequence

from . import capi
from .capi import AttentionDesc, DCNv2Error, DType, Norm, RotaryDesc, Status, lib


@functools.lru_cache(maxsize=None)
def _dtypes():
    import torch
    return {torch.float32: int(DType.FLOAT), torch.float16: int(DType.HALF),
            torch.bfloat16: int(DType.BF16)}


@contextlib.contextmanager
def _on(device, stream):
    """`device` current, and allocations made for `stream` (a raw handle; None: the current one)."""
    import torch
    with torch.cuda.device(device):
        if stream is None:
            yield torch.cuda.current_stream(device).cuda_stream
        else:
            with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device)):
                yield stream


def _check(what, name, t, dtype, device, ndim):
    if t.dtype != dtype:
        raise TypeError(f"{what}: {name} is {t.dtype}, expected {dtype}")
    if t.dim() != ndim:
        raise ValueError(f"{what}: {name} has {t.dim()} dimensions, expected {ndim}")
    if not t.is_cuda or t.device != device:
        raise ValueError(f"{what}: {name} is not on {device}")


def _check_heads(what, name, t, dtype, device):
    _check(what, name, t, dtype, device, 4)
    if t.shape[3] > 1 and t.stride(3) != 1:
        raise ValueError(f"{what}: the elements of a head of {name} are not contiguous")


def rotary_axes(rotary_dim: int, sections: Sequence[int], base: float = 10000.0,
                turns: bool = False, shared_table: bool = False, device="cuda"):
    """(freqs, pair_axis) of dcnv2_qk_norm_rotary for a rotary_dim of which sections[i] pairs turn by
    axis i. turns=False: the axes one after another; True: in turn (0, 1, 2, 0, 1, ...), an axis
    dropping out when its pairs are used up. shared_table=True: pair p of all has frequency
    base^(-2p/rotary_dim); False: each axis has the table base^(-j/sections[i]) of its own pairs."""
    import torch
    if rotary_dim < 2 or rotary_dim % 2 or not 1 <= len(sections) <= 4 or \
            any(n < 0 for n in sections) or sum(sections) != rotary_dim // 2:
        raise ValueError("rotary_axes: one to four sections that add up to rotary_dim / 2 pairs")
    if turns:
        axes, left = [], list(sections)
        while len(axes) < rotary_dim // 2:
            for i, n in enumerate(left):
                if n:
                    axes.append(i)
                    left[i] -= 1
    else:
        axes = [i for i, n in enumerate(sections) for _ in range(n)]
    if shared_table:
        freqs = [base ** (-2.0 * p / rotary_dim) for p in range(rotary_dim // 2)]
    else:
        freqs = [base ** (-axes[:p].count(a) / sections[a]) for p, a in enumerate(axes)]
    return torch.tensor(freqs, dtype=torch.float32, device=device), bytes(axes)


def level_positions(sizes: Sequence[Sequence[int]], device="cuda"):
    """int32 [1, sum of h * w, 3]: (level, row, column) of every pixel of maps of the given (h, w), in
    the order of the maps and row by row, for dcnv2_qk_norm_rotary with three axes."""
    import torch
    parts = []
    for level, (h, w) in enumerate(sizes):
        i = torch.arange(h * w, dtype=torch.int32)
        parts.append(torch.stack([torch.full_like(i, level),
                                  torch.div(i, w, rounding_mode="floor"), i % w], 1))
    if not parts:
        raise ValueError("level_positions needs at least one map")
    return torch.cat(parts)[None].contiguous().to(device)


@functools.lru_cache(maxsize=1024)
def _rotary_desc(batch, tokens, q_heads, k_heads, head_dim, rotary_dim, axes, dtype, norm,
                 interleaved, eps, pair_axis, strides, pos_batch_stride):
    d = RotaryDesc(batch, tokens, q_heads, k_heads, head_dim, rotary_dim, axes, dtype, norm,
                   interleaved, eps)
    ctypes.memmove(d.pair_axis, pair_axis, len(pair_axis))
    for field, st in zip((d.q_stride, d.k_stride, d.q_out_stride, d.k_out_stride), strides):
        field[:] = st
    d.pos_batch_stride = pos_batch_stride
    return d


def dcnv2_qk_norm_rotary(q, k=None, positions=None, freqs=None, pair_axis=b"", q_weight=None,
                         k_weight=None, norm=None, eps: float = 1e-6, interleaved: bool = False,
                         q_out=None, k_out=None, stream=None):
    """(q', k'): each head normalised (norm="rms": x * rsqrt(mean(x^2) + eps) * weight) and rotated
    by its token's position.

    q, k       [batch, tokens, heads, head_dim] fp32, fp16 or bf16, one of them may be None; any
               strides with contiguous heads; head_dim even, at most 256
    positions  int32 [batch or 1, tokens, axes] (or [tokens, axes]), contiguous
    freqs, pair_axis  fp32 [pairs] and the axis of each pair (rotary_axes makes both); the first
               2 * pairs elements of a head are rotated (none without them)
    q_weight, k_weight  [head_dim] gains of the norm, of q's dtype, or None (ones)
    q_out, k_out  outputs; q and k themselves rotate in place
    Returns contiguous tensors unless outputs are given; None stands for an absent one."""
    import torch
    what = "dcnv2_qk_norm_rotary"
    x = q if q is not None else k
    if x is None:
        raise ValueError(f"{what}: q or k is needed")
    if x.dtype not in _dtypes():
        raise TypeError(f"{what}: unsupported dtype {x.dtype}")
    if norm not in (None, "rms"):
        raise ValueError(f"{what}: norm is None or 'rms'")
    dt, dev = x.dtype, x.device
    B, T, D = x.shape[0], x.shape[1], x.shape[-1]
    outs = []
    for name, t, o, w in (("q", q, q_out, q_weight), ("k", k, k_out, k_weight)):
        if t is None:
            if o is not None or w is not None:
                raise ValueError(f"{what}: {name}_out or {name}_weight without {name}")
            continue
        _check_heads(what, name, t, dt, dev)
        if (t.shape[0], t.shape[1], t.shape[3]) != (B, T, D):
            raise ValueError(f"{what}: q and k differ in batch, tokens or head_dim")
        if o is not None:
            _check_heads(what, f"{name}_out", o, dt, dev)
            if o.shape != t.shape:
                raise ValueError(f"{what}: {name}_out has another shape than {name}")
        if w is not None:
            _check(what, f"{name}_weight", w, dt, dev, 1)
            if w.shape[0] != D or not w.is_contiguous():
                raise ValueError(f"{what}: {name}_weight is not a contiguous [{D}]")
            if norm is None:
                raise ValueError(f"{what}: {name}_weight without norm='rms'")
    pairs, axes, pos_sb = 0, 1, 0
    if freqs is not None:
        pair_axis = bytes(pair_axis)
        pairs = len(pair_axis)
        _check(what, "freqs", freqs, torch.float32, dev, 1)
        if freqs.shape[0] != pairs or not freqs.is_contiguous() or 2 * pairs > D or pairs > 128:
            raise ValueError(f"{what}: freqs and pair_axis give one value for each of at most "
                             f"{min(D // 2, 128)} rotated pairs")
        if positions is None:
            raise ValueError(f"{what}: rotation needs positions")
        if positions.dim() == 2:
            positions = positions[None]
        _check(what, "positions", positions, torch.int32, dev, 3)
        if positions.shape[0] not in (1, B) or positions.shape[1] != T or \
                not positions.is_contiguous():
            raise ValueError(f"{what}: positions are not a contiguous [{B} or 1, {T}, axes]")
        axes = positions.shape[2]
        pos_sb = T * axes if positions.shape[0] > 1 else 0
    elif positions is not None or len(pair_axis):
        raise ValueError(f"{what}: positions or pair_axis without freqs")
    same = stream is None and dev.index == torch.cuda.current_device()
    with contextlib.nullcontext() if same else _on(dev, stream) as st:
        if same:
            st = torch.cuda.current_stream().cuda_stream
        if q is not None and q_out is None:
            q_out = torch.empty(q.shape, dtype=dt, device=dev)
        if k is not None and k_out is None:
            k_out = torch.empty(k.shape, dtype=dt, device=dev)
        strides = tuple(t.stride()[:3] if t is not None else (0, 0, 0)
                        for t in (q, k, q_out, k_out))
        desc = _rotary_desc(B, T, q.shape[2] if q is not None else 0,
                            k.shape[2] if k is not None else 0, D, 2 * pairs, axes,
                            _dtypes()[dt], int(Norm.RMS if norm else Norm.NONE), int(interleaved),
                            float(eps), pair_axis, strides, pos_sb)
        if x.numel() == 0 and (k is None or k.numel() == 0):
            return q_out, k_out
        rc = lib.dcnv2_qk_norm_rotary(
            ctypes.byref(desc), *(t.data_ptr() if t is not None else None for t in (
                q, k, positions, freqs, q_weight, k_weight, q_out, k_out)), st)
    if rc != Status.OK:
        raise DCNv2Error(rc, what)
    return q_out, k_out


@functools.lru_cache(maxsize=1024)
def _attention_desc(batch, q_tokens, kv_tokens, q_heads, kv_heads, head_dim, dtype, scale, strides,
                    mask_batch_stride):
    """The desc and its workspace size."""
    d = AttentionDesc(batch, q_tokens, kv_tokens, q_heads, kv_heads, head_dim, dtype, scale)
    for field, st in zip((d.q_stride, d.k_stride, d.v_stride, d.out_stride), strides):
        field[:] = st
    d.mask_batch_stride = mask_batch_stride
    return d, int(lib.dcnv2_cross_attention_workspace_size(ctypes.byref(d)))


def _legal_strides(t):
    """Batch, token and head strides; of a dimension that takes no step, 0."""
    return tuple(s if n > 1 else 0 for s, n in zip(t.stride(), t.shape[:3]))


def dcnv2_cross_attention(q, k, v, kv_lens=None, key_mask=None, scale=None,
                          return_lse: bool = False, out=None, workspace=None, stream=None):
    """out = softmax(scale * q k^T over the kept states) v, queries of one sequence over the states
    of another.

    q          [batch, q_tokens, q_heads, head_dim] fp16 or bf16; one token or many
    k, v       [batch, kv_tokens, kv_heads, head_dim]; q_heads a multiple of kv_heads; expanded
               (shared) batches are read in place
    kv_lens    int32 [batch]: kept states per sequence; None keeps all
    key_mask   bool or uint8 [batch or 1, kv_tokens]: states kept (pixels of padded images)
    scale      of the scores; None: 1 / sqrt(head_dim)
    workspace  uint8 CUDA tensor of at least dcnv2_cross_attention_workspace_size bytes (allocated
               when absent or too small); not shared by calls that may overlap
    All tensors: any strides that are multiples of 8 elements, contiguous heads, 16-byte aligned;
    head_dim a multiple of 8, at most 128. A sequence without kept states gives zeros. Returns out
    [batch, q_tokens, q_heads, head_dim], or (out, lse) with lse fp32 [batch, q_heads, q_tokens]."""
    import torch
    what = "dcnv2_cross_attention"
    dt, dev = q.dtype, q.device
    if dt not in (torch.float16, torch.bfloat16):
        raise TypeError(f"{what}: unsupported dtype {dt}")
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check_heads(what, name, t, dt, dev)
    B, L, H, D = q.shape
    S, G = k.shape[1], k.shape[2]
    if k.shape[0] != B or k.shape[3] != D or v.shape != k.shape:
        raise ValueError(f"{what}: k and v are not [{B}, kv_tokens, kv_heads, {D}]")
    if out is not None:
        _check_heads(what, "out", out, dt, dev)
        if out.shape != q.shape:
            raise ValueError(f"{what}: out has another shape than q")
    if kv_lens is not None:
        _check(what, "kv_lens", kv_lens, torch.int32, dev, 1)
        if kv_lens.shape[0] != B or not kv_lens.is_contiguous():
            raise ValueError(f"{what}: kv_lens is not a contiguous [{B}]")
    mask_sb = 0
    if key_mask is not None:
        if key_mask.dtype not in (torch.bool, torch.uint8):
            raise TypeError(f"{what}: key_mask is bool or uint8")
        _check(what, "key_mask", key_mask, key_mask.dtype, dev, 2)
        if key_mask.shape[0] not in (1, B) or key_mask.shape[1] != S or \
                (S > 1 and key_mask.stride(1) != 1):
            raise ValueError(f"{what}: key_mask is not [{B} or 1, {S}] with contiguous rows")
        mask_sb = key_mask.stride(0) if key_mask.shape[0] > 1 else 0
    if scale is None:
        scale = 1.0 / math.sqrt(D) if D else 1.0
    if workspace is not None and (not workspace.is_cuda or workspace.device != dev):
        raise ValueError(f"{what}: workspace is not on {dev}")
    same = stream is None and dev.index == torch.cuda.current_device()
    with contextlib.nullcontext() if same else _on(dev, stream) as st:
        if same:
            st = torch.cuda.current_stream().cuda_stream
        if out is None:
            out = torch.empty(q.shape, dtype=dt, device=dev)
        lse = torch.empty((B, H, L), dtype=torch.float32, device=dev) if return_lse else None
        if out.numel() == 0:
            return (out, lse) if return_lse else out
        desc, ws_bytes = _attention_desc(
            B, L, S, H, G, D, _dtypes()[dt], float(scale),
            tuple(_legal_strides(t) for t in (q, k, v, out)), mask_sb)
        if workspace is None or workspace.numel() < ws_bytes:
            workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        rc = lib.dcnv2_cross_attention(
            ctypes.byref(desc), *(t.data_ptr() if t is not None else None for t in (
                q, k, v, kv_lens, key_mask, out, lse, workspace)), workspace.numel(), st)
    if rc != Status.OK:
        raise DCNv2Error(rc, what)
    return (out, lse) if return_lse else out
