"""Token operators on the layer's feature maps, backed by libdcnv2.so: what a transformer that
reads the maps (a detection decoder, a language model with image tokens) does with them.

dcnv2_qk_norm_rotary   RMS norm of each query and key head and its rotation by the token's position
                       on one to four axes (text; row and column; frame or level, row, column)
dcnv2_cross_attention  attention of queries to the states of another sequence: many queries or
                       single tokens, grouped heads, lengths and masks of padded images
dcnv2_cross_attention_workspace_size, dcnv2_cross_attention_error
                       the workspace of such a call, and the error words that it left there
rotary_axes            frequency table and axis of each rotated pair, made once per model
level_positions        (level, row, column) of every pixel of a pyramid's levels

Both operators take strided torch CUDA tensors (views of one projection, caches laid out heads
first), run on the current torch stream of the tensors' device unless a stream is given, and raise
DCNv2Error when the call is refused or cannot be launched. A wait inside the attention's kernel that
runs out later makes the rows it concerns NaN; who wants to be told keeps the workspace and reads its
error words (dcnv2_cross_attention_error). They are inference operators, as the layer is: no gradients.
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


# Calls of these operators take a few microseconds on the GPU, so what depends on the arguments' shapes,
# strides, types and devices alone (the checks, the desc) is done once for each combination and kept
# under those values. A tensor is described by:
def _meta(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())


@contextlib.contextmanager
def _on(index, stream):
    """Device `index` current, and allocations made for `stream` (a raw handle; None: the current
    one); gives the raw handle."""
    import torch
    with torch.cuda.device(index):
        if stream is None:
            yield torch.cuda.current_stream(index).cuda_stream
        else:
            with torch.cuda.stream(torch.cuda.ExternalStream(stream,
                                                             device=torch.device("cuda", index))):
                yield stream


def _current(index):
    """The raw handle of the current stream of device `index` if that device is current, else None."""
    import torch
    if torch.cuda.current_device() != index:
        return None
    return torch._C._cuda_getCurrentRawStream(index)


def _check(what, name, meta, dtype, index, ndim):
    shape, _, dt, on = meta
    if dt != dtype:
        raise TypeError(f"{what}: {name} is {dt}, expected {dtype}")
    if len(shape) != ndim:
        raise ValueError(f"{what}: {name} has {len(shape)} dimensions, expected {ndim}")
    if on < 0 or on != index:
        raise ValueError(f"{what}: {name} is not on cuda:{index}")


def _check_heads(what, name, meta, dtype, index):
    _check(what, name, meta, dtype, index, 4)
    if meta[0][3] > 1 and meta[1][3] != 1:
        raise ValueError(f"{what}: the elements of a head of {name} are not contiguous")


def _contiguous(shape, strides):
    step = 1
    for n, st in zip(reversed(shape), reversed(strides)):
        if n > 1 and st != step:
            return 0 in shape
        step *= n
    return True


def _packed(shape):
    """Batch, token and head strides of a contiguous tensor."""
    _, t, h, d = shape
    return t * h * d, h * d, d


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
def _rotary_plan(q, k, q_out, k_out, positions, freqs, q_weight, k_weight, pair_axis, norm, eps,
                 interleaved):
    """Checks the metas; (desc, device index, whether there is nothing to do)."""
    import torch
    what = "dcnv2_qk_norm_rotary"
    x = q or k
    if x is None:
        raise ValueError(f"{what}: q or k is needed")
    shape, _, dt, index = x
    if dt not in _dtypes():
        raise TypeError(f"{what}: unsupported dtype {dt}")
    if norm not in (None, "rms"):
        raise ValueError(f"{what}: norm is None or 'rms'")
    for name, t, o, w in (("q", q, q_out, q_weight), ("k", k, k_out, k_weight)):
        if t is None:
            if o is not None or w is not None:
                raise ValueError(f"{what}: {name}_out or {name}_weight without {name}")
            continue
        _check_heads(what, name, t, dt, index)
        if (t[0][0], t[0][1], t[0][3]) != (shape[0], shape[1], shape[3]):
            raise ValueError(f"{what}: q and k differ in batch, tokens or head_dim")
        if o is not None:
            _check_heads(what, f"{name}_out", o, dt, index)
            if o[0] != t[0]:
                raise ValueError(f"{what}: {name}_out has another shape than {name}")
        if w is not None:
            _check(what, f"{name}_weight", w, dt, index, 1)
            if w[0][0] != shape[3] or not _contiguous(w[0], w[1]):
                raise ValueError(f"{what}: {name}_weight is not a contiguous [{shape[3]}]")
            if norm is None:
                raise ValueError(f"{what}: {name}_weight without norm='rms'")
    B, T, _, D = shape
    pairs, axes, pos_sb = 0, 1, 0
    if freqs is not None:
        pairs = len(pair_axis)
        _check(what, "freqs", freqs, torch.float32, index, 1)
        if freqs[0][0] != pairs or not _contiguous(freqs[0], freqs[1]) or 2 * pairs > D or \
                pairs > 128:
            raise ValueError(f"{what}: freqs and pair_axis give one value for each of at most "
                             f"{min(D // 2, 128)} rotated pairs")
        if positions is None:
            raise ValueError(f"{what}: rotation needs positions")
        if len(positions[0]) == 2:
            positions = ((1,) + tuple(positions[0]), (0,) + tuple(positions[1])) + positions[2:]
        _check(what, "positions", positions, torch.int32, index, 3)
        (n, tokens, axes), strides = positions[0], positions[1]
        if n not in (1, B) or tokens != T or not _contiguous(positions[0], strides):
            raise ValueError(f"{what}: positions are not a contiguous [{B} or 1, {T}, axes]")
        pos_sb = T * axes if n > 1 else 0
    elif positions is not None or len(pair_axis):
        raise ValueError(f"{what}: positions or pair_axis without freqs")
    d = RotaryDesc(B, T, q[0][2] if q else 0, k[0][2] if k else 0, D, 2 * pairs, axes,
                   _dtypes()[dt], int(Norm.RMS if norm else Norm.NONE), int(interleaved), eps)
    ctypes.memmove(d.pair_axis, pair_axis, len(pair_axis))
    for t, o, field, out_field in ((q, q_out, d.q_stride, d.q_out_stride),
                                   (k, k_out, d.k_stride, d.k_out_stride)):
        if t is not None:
            field[:] = t[1][:3]
            out_field[:] = o[1][:3] if o is not None else _packed(t[0])
    d.pos_batch_stride = pos_sb
    # (a reference to d keeps it)
    return ctypes.byref(d), index, 0 in (B, T, D) or not (d.q_heads or d.k_heads)


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
    desc, index, nothing = _rotary_plan(
        _meta(q), _meta(k), _meta(q_out), _meta(k_out), _meta(positions), _meta(freqs),
        _meta(q_weight), _meta(k_weight), bytes(pair_axis), norm, float(eps), bool(interleaved))
    st = _current(index) if stream is None else None
    if st is None:
        with _on(index, stream) as st:
            return _rotary_launch(desc, nothing, q, k, positions, freqs, q_weight, k_weight, q_out,
                                  k_out, st)
    return _rotary_launch(desc, nothing, q, k, positions, freqs, q_weight, k_weight, q_out, k_out, st)


def _rotary_launch(desc, nothing, q, k, positions, freqs, q_weight, k_weight, q_out, k_out, st):
    import torch
    if q is not None and q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if k is not None and k_out is None:
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    if nothing:
        return q_out, k_out
    rc = lib.dcnv2_qk_norm_rotary(
        desc, q if q is None else q.data_ptr(), k if k is None else k.data_ptr(),
        positions if positions is None else positions.data_ptr(),
        freqs if freqs is None else freqs.data_ptr(),
        q_weight if q_weight is None else q_weight.data_ptr(),
        k_weight if k_weight is None else k_weight.data_ptr(),
        q_out if q_out is None else q_out.data_ptr(), k_out if k_out is None else k_out.data_ptr(),
        st)
    if rc:
        raise DCNv2Error(rc, "dcnv2_qk_norm_rotary")
    return q_out, k_out


@functools.lru_cache(maxsize=1024)
def _attention_plan(q, k, v, out, kv_lens, key_mask, scale):
    """Checks the metas; (desc, workspace bytes, device index, shape of lse, whether there is nothing
    to do)."""
    import torch
    what = "dcnv2_cross_attention"
    (B, L, H, D), _, dt, index = q if len(q[0]) == 4 else ((0, 0, 0, 0),) + q[1:]
    if dt not in (torch.float16, torch.bfloat16):
        raise TypeError(f"{what}: unsupported dtype {dt}")
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check_heads(what, name, t, dt, index)
    _, S, G, _ = k[0]
    if k[0][0] != B or k[0][3] != D or v[0] != k[0]:
        raise ValueError(f"{what}: k and v are not [{B}, kv_tokens, kv_heads, {D}]")
    if out is not None:
        _check_heads(what, "out", out, dt, index)
        if out[0] != q[0]:
            raise ValueError(f"{what}: out has another shape than q")
    if kv_lens is not None:
        _check(what, "kv_lens", kv_lens, torch.int32, index, 1)
        if kv_lens[0][0] != B or not _contiguous(kv_lens[0], kv_lens[1]):
            raise ValueError(f"{what}: kv_lens is not a contiguous [{B}]")
    mask_sb = 0
    if key_mask is not None:
        if key_mask[2] not in (torch.bool, torch.uint8):
            raise TypeError(f"{what}: key_mask is bool or uint8")
        _check(what, "key_mask", key_mask, key_mask[2], index, 2)
        if key_mask[0][0] not in (1, B) or key_mask[0][1] != S or (S > 1 and key_mask[1][1] != 1):
            raise ValueError(f"{what}: key_mask is not [{B} or 1, {S}] with contiguous rows")
        mask_sb = key_mask[1][0] if key_mask[0][0] > 1 else 0
    if scale is None:
        scale = 1.0 / math.sqrt(D) if D else 1.0
    d = AttentionDesc(B, L, S, H, G, D, _dtypes()[dt], scale)
    for field, shape, strides in ((d.q_stride, q[0], q[1]), (d.k_stride, k[0], k[1]),
                                  (d.v_stride, v[0], v[1]),
                                  (d.out_stride, q[0], out[1] if out else _packed(q[0]))):
        # of a dimension that takes no step, 0
        field[:] = tuple(st if n > 1 else 0 for st, n in zip(strides, shape[:3]))
    d.mask_batch_stride = mask_sb
    nothing = 0 in (B, L, H, D)
    # (a reference to d keeps it)
    return (ctypes.byref(d), 0 if nothing else capi.attention_workspace_size(d), index, (B, H, L),
            nothing)


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
    workspace  contiguous CUDA tensor of at least dcnv2_cross_attention_workspace_size(q, k, v) bytes
               (allocated when absent or too small, and dropped with its error words); not shared by
               calls that may overlap
    All tensors: any strides that are multiples of 8 elements, contiguous heads, 16-byte aligned;
    head_dim a multiple of 8, at most 128. A sequence without kept states gives zeros. Returns out
    [batch, q_tokens, q_heads, head_dim], or (out, lse) with lse fp32 [batch, q_heads, q_tokens]."""
    import torch
    desc, ws_bytes, index, lse_shape, nothing = _attention_plan(
        _meta(q), _meta(k), _meta(v), _meta(out), _meta(kv_lens), _meta(key_mask),
        None if scale is None else float(scale))
    if workspace is not None and (workspace.get_device() != index or
                                  not workspace.is_contiguous()):
        raise ValueError(f"dcnv2_cross_attention: workspace is not a contiguous tensor on cuda:{index}")
    st = _current(index) if stream is None else None
    if st is None:
        with _on(index, stream) as st:
            out, lse = _attention_launch(desc, ws_bytes, nothing, q, k, v, kv_lens, key_mask, out,
                                         lse_shape if return_lse else None, workspace, st)
    else:
        out, lse = _attention_launch(desc, ws_bytes, nothing, q, k, v, kv_lens, key_mask, out,
                                     lse_shape if return_lse else None, workspace, st)
    return (out, lse) if return_lse else out


def _attention_launch(desc, ws_bytes, nothing, q, k, v, kv_lens, key_mask, out, lse_shape, workspace,
                      st):
    import torch
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = q.new_empty(lse_shape, dtype=torch.float32) if lse_shape is not None else None
    if nothing:
        return out, lse
    if ws_bytes and (workspace is None or workspace.nbytes < ws_bytes):
        workspace = q.new_empty((ws_bytes,), dtype=torch.uint8)
    rc = lib.dcnv2_cross_attention(
        desc, q.data_ptr(), k.data_ptr(), v.data_ptr(),
        kv_lens if kv_lens is None else kv_lens.data_ptr(),
        key_mask if key_mask is None else key_mask.data_ptr(), out.data_ptr(),
        lse if lse is None else lse.data_ptr(),
        workspace if workspace is None else workspace.data_ptr(), ws_bytes, st)
    if rc:
        raise DCNv2Error(rc, "dcnv2_cross_attention")
    return out, lse


def dcnv2_cross_attention_workspace_size(q, k, v) -> int:
    """Workspace bytes of dcnv2_cross_attention(q, k, v): one error word per CTA, or 0 when nothing in
    the call waits (up to 16 query rows per kv head) or there is nothing to do."""
    return _attention_plan(_meta(q), _meta(k), _meta(v), None, None, None, None)[1]


def dcnv2_cross_attention_error(q, k, v, workspace, stream=None) -> int:
    """Error bits (0: none) that the last dcnv2_cross_attention call with tensors of these shapes and
    strides left in the workspace it was given, after synchronising the stream (the current one of q's
    device unless given). Not during a stream capture."""
    what = "dcnv2_cross_attention_error"
    desc, ws_bytes, index, _, _ = _attention_plan(_meta(q), _meta(k), _meta(v), None, None, None, None)
    if ws_bytes == 0:
        return 0
    if workspace is None or workspace.get_device() != index or not workspace.is_contiguous() or \
            workspace.nbytes < ws_bytes:
        raise ValueError(f"{what}: workspace is not a contiguous tensor of {ws_bytes} bytes on "
                         f"cuda:{index}")
    code = ctypes.c_int32(0)
    with _on(index, stream) as st:
        rc = lib.dcnv2_cross_attention_read_error(desc, workspace.data_ptr(), st, ctypes.byref(code))
    if rc not in (Status.OK, Status.ERR_DEVICE_TIMEOUT):
        raise DCNv2Error(rc, what)
    return code.value
