"""Host-side checks of the token operators that need no GPU: the refusals of the C entry points (made
before a device is asked for), workspace sizes, and the tables rotary_axes and level_positions make."""
import ctypes

import pytest
import torch

from dcnv2_b200 import capi, level_positions, rotary_axes
from dcnv2_b200.capi import DType, Status, lib

P = 0x10000  # an aligned address; nothing here launches


def rotary_desc(**kw):
    a = dict(batch=2, tokens=3, q_heads=4, k_heads=2, head_dim=64, rotary_dim=64, axes=2,
             dtype=int(DType.HALF), norm=1, interleaved=0, eps=1e-6, pair_axis=[0, 1] * 16)
    a.update(kw)
    axis, strides = a.pop("pair_axis"), a.pop("strides", {})
    d = capi.RotaryDesc(**a)
    for i, x in enumerate(axis):
        d.pair_axis[i] = x
    for n, h in (("q", a["q_heads"]), ("k", a["k_heads"])):
        st = (a["tokens"] * h * a["head_dim"], h * a["head_dim"], a["head_dim"])
        getattr(d, f"{n}_stride")[:] = strides.get(n, st)
        getattr(d, f"{n}_out_stride")[:] = strides.get(f"{n}_out", st)
    d.pos_batch_stride = strides.get("pos", 6)
    return d


def rotary(d, q=P, k=P, pos=P, freqs=P, qw=P, kw=P, qo=P, ko=P):
    return lib.dcnv2_qk_norm_rotary(ctypes.byref(d) if d is not None else None, q, k, pos, freqs, qw,
                                    kw, qo, ko, None)


@pytest.mark.parametrize("kw,status", [
    (dict(batch=-1), Status.ERR_INVALID_ARG),
    (dict(tokens=-1), Status.ERR_INVALID_ARG),
    (dict(q_heads=-1), Status.ERR_INVALID_ARG),
    (dict(q_heads=0, k_heads=0), Status.ERR_INVALID_ARG),
    (dict(q_heads=65536, k_heads=1), Status.ERR_INVALID_ARG),
    (dict(batch=65536, tokens=65536), Status.ERR_INVALID_ARG),
    (dict(head_dim=63), Status.ERR_INVALID_ARG),
    (dict(head_dim=0), Status.ERR_INVALID_ARG),
    (dict(head_dim=258), Status.ERR_UNSUPPORTED),
    (dict(rotary_dim=66), Status.ERR_INVALID_ARG),
    (dict(rotary_dim=31), Status.ERR_INVALID_ARG),
    (dict(rotary_dim=-2), Status.ERR_INVALID_ARG),
    (dict(axes=0), Status.ERR_INVALID_ARG),
    (dict(axes=5), Status.ERR_INVALID_ARG),
    (dict(axes=1), Status.ERR_INVALID_ARG),                  # pair_axis names axis 1
    (dict(pair_axis=[0, 255] * 16), Status.ERR_INVALID_ARG),
    (dict(dtype=int(DType.INT8)), Status.ERR_UNSUPPORTED),
    (dict(dtype=99), Status.ERR_UNSUPPORTED),
    (dict(norm=2), Status.ERR_INVALID_ARG),
    (dict(eps=-1.0), Status.ERR_INVALID_ARG),
    (dict(eps=float("nan")), Status.ERR_INVALID_ARG),
    (dict(interleaved=2), Status.ERR_INVALID_ARG),
    (dict(strides={"q": (-1, 256, 64)}), Status.ERR_INVALID_ARG),
    (dict(strides={"k": (1 << 61, 128, 64)}), Status.ERR_INVALID_ARG),
    (dict(strides={"q_out": (0, 256, 64)}), Status.ERR_INVALID_ARG),  # rows over one another
    (dict(strides={"k_out": (384, 128, 32)}), Status.ERR_INVALID_ARG),
    (dict(strides={"pos": -6}), Status.ERR_INVALID_ARG),
])
def test_rotary_refusals(kw, status):
    assert rotary(rotary_desc(**kw)) == status


def test_rotary_pointer_refusals_and_no_ops():
    bad = Status.ERR_INVALID_ARG
    assert rotary(None) == bad
    for null in ("q", "k", "pos", "freqs", "qo", "ko"):
        assert rotary(rotary_desc(), **{null: None}) == bad
    assert rotary(rotary_desc(), q=P + 1) == bad            # not aligned to an element
    assert rotary(rotary_desc(), pos=P + 2) == bad
    assert rotary(rotary_desc(batch=0), q=None, k=None) == Status.OK
    assert rotary(rotary_desc(tokens=0)) == Status.OK
    if not torch.cuda.is_available():
        assert rotary(rotary_desc()) == Status.ERR_NO_DEVICE
        assert rotary(rotary_desc(k_heads=0), k=None, ko=None) == Status.ERR_NO_DEVICE
        assert rotary(rotary_desc(rotary_dim=0, axes=0), pos=None, freqs=None,
                      qw=None, kw=None) == Status.ERR_NO_DEVICE


def attention_desc(**kw):
    a = dict(batch=2, q_tokens=5, kv_tokens=300, q_heads=8, kv_heads=2, head_dim=64,
             dtype=int(DType.BF16), scale=0.125)
    a.update(kw)
    strides = a.pop("strides", {})
    d = capi.AttentionDesc(**a)
    for n, t, h in (("q", a["q_tokens"], a["q_heads"]), ("k", a["kv_tokens"], a["kv_heads"]),
                    ("v", a["kv_tokens"], a["kv_heads"]), ("out", a["q_tokens"], a["q_heads"])):
        st = (t * h * a["head_dim"], h * a["head_dim"], a["head_dim"])
        getattr(d, f"{n}_stride")[:] = strides.get(n, st)
    d.mask_batch_stride = strides.get("mask", a["kv_tokens"])
    return d


def attention(d, q=P, k=P, v=P, lens=None, mask=None, out=P, lse=P, ws=P, ws_bytes=1 << 20):
    return lib.dcnv2_cross_attention(ctypes.byref(d) if d is not None else None, q, k, v, lens, mask,
                                     out, lse, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,status", [
    (dict(batch=-1), Status.ERR_INVALID_ARG),
    (dict(q_tokens=-1), Status.ERR_INVALID_ARG),
    (dict(kv_tokens=-1), Status.ERR_INVALID_ARG),
    (dict(q_heads=0), Status.ERR_INVALID_ARG),
    (dict(kv_heads=0), Status.ERR_INVALID_ARG),
    (dict(kv_heads=3), Status.ERR_INVALID_ARG),
    (dict(head_dim=0), Status.ERR_INVALID_ARG),
    (dict(head_dim=60), Status.ERR_UNSUPPORTED),
    (dict(head_dim=136), Status.ERR_UNSUPPORTED),
    (dict(dtype=int(DType.FLOAT)), Status.ERR_UNSUPPORTED),
    (dict(dtype=int(DType.INT8)), Status.ERR_UNSUPPORTED),
    (dict(scale=0.0), Status.ERR_INVALID_ARG),
    (dict(scale=-1.0), Status.ERR_INVALID_ARG),
    (dict(scale=float("inf")), Status.ERR_INVALID_ARG),
    (dict(scale=float("nan")), Status.ERR_INVALID_ARG),
    (dict(strides={"q": (2560, 516, 64)}), Status.ERR_UNSUPPORTED),
    (dict(strides={"v": (38400, 128, 68)}), Status.ERR_UNSUPPORTED),
    (dict(strides={"k": (-8, 128, 64)}), Status.ERR_INVALID_ARG),
    (dict(strides={"out": (0, 512, 64)}), Status.ERR_INVALID_ARG),
    (dict(strides={"q": (2560, 0, 64)}), Status.ERR_UNSUPPORTED),   # shared along tokens, heads
    (dict(strides={"q": (2560, 512, 0)}), Status.ERR_UNSUPPORTED),
    (dict(strides={"k": (38400, 0, 64)}), Status.ERR_UNSUPPORTED),
    (dict(kv_tokens=2 ** 31 - 1), Status.ERR_INVALID_ARG),
    (dict(strides={"mask": -300}), Status.ERR_INVALID_ARG),
    (dict(batch=1 << 20, q_tokens=1 << 20), Status.ERR_INVALID_ARG),
])
def test_attention_refusals(kw, status):
    d = attention_desc(**kw)
    assert attention(d) == status
    assert lib.dcnv2_cross_attention_workspace_size(ctypes.byref(d)) == 0


@pytest.mark.parametrize("strides", [
    (256, 64, 64),        # tokens and heads in the same places
    (768, 128, 64),       # four heads of 64 in 128
    (512, 256, 64),       # three tokens of 256 in 512
    (64, 384, 128),       # sequences inside a head's step, tokens inside the heads' reach
])
def test_outputs_over_themselves_are_refused(strides):
    assert rotary(rotary_desc(strides={"q_out": strides})) == Status.ERR_INVALID_ARG
    d = attention_desc(q_tokens=3, q_heads=4, strides={"out": strides})
    assert attention(d) == Status.ERR_INVALID_ARG


def test_outputs_in_other_orders_are_taken():
    if torch.cuda.is_available():
        pytest.skip("would launch")
    for strides in ((4 * 3 * 64, 64, 3 * 64),     # heads first
                    (64, 4 * 2 * 64, 2 * 64),     # tokens, heads, sequences
                    (4096, 1024, 72)):            # gaps
        assert rotary(rotary_desc(strides={"q_out": strides})) == Status.ERR_NO_DEVICE
        d = attention_desc(q_tokens=3, q_heads=4, strides={"out": strides})
        assert attention(d) == Status.ERR_NO_DEVICE
    d = attention_desc(q_tokens=1, q_heads=4, strides={"out": (256, 0, 64)})  # a step never taken
    assert attention(d) == Status.ERR_NO_DEVICE


def test_attention_scale_and_masked_length_limits():
    assert attention(attention_desc(scale=3e38)) == Status.ERR_INVALID_ARG  # infinite in base 2
    long = dict(batch=1, q_tokens=200, q_heads=2, kv_heads=2, head_dim=8, kv_tokens=(1 << 28) + 1)
    assert attention(attention_desc(**long), mask=P) == Status.ERR_UNSUPPORTED
    if not torch.cuda.is_available():
        assert attention(attention_desc(**long)) == Status.ERR_NO_DEVICE
        long["kv_tokens"] -= 1
        assert attention(attention_desc(**long), mask=P) == Status.ERR_NO_DEVICE


def test_attention_pointer_refusals_and_no_ops():
    d = attention_desc()
    bad = Status.ERR_INVALID_ARG
    assert attention(None) == bad
    assert lib.dcnv2_cross_attention_workspace_size(None) == 0
    for null in ("q", "k", "v", "out"):
        assert attention(d, **{null: None}) == bad
        assert attention(d, **{null: P + 8}) == Status.ERR_UNSUPPORTED  # 16-byte alignment
    assert attention(d, lens=P + 1) == bad and attention(d, lse=P + 2) == bad
    need = lib.dcnv2_cross_attention_workspace_size(ctypes.byref(d))
    assert 0 < need <= 1 << 20
    assert attention(d, ws=None) == Status.ERR_WORKSPACE
    assert attention(d, ws=P + 2) == Status.ERR_WORKSPACE
    assert attention(d, ws_bytes=0) == Status.ERR_WORKSPACE
    few = attention_desc(q_tokens=1)  # no workspace for up to 16 rows per kv head
    assert lib.dcnv2_cross_attention_workspace_size(ctypes.byref(few)) == 0
    assert attention(attention_desc(batch=0)) == Status.OK
    assert attention(attention_desc(q_tokens=0), q=None, out=None) == Status.OK
    if not torch.cuda.is_available():
        assert attention(d, lse=None, mask=P + 1) == Status.ERR_NO_DEVICE
        assert attention(d, ws_bytes=need) == Status.ERR_NO_DEVICE
        # strides that no step is taken by may hold anything
        one = attention_desc(batch=1, q_tokens=1, strides={"q": (3, 5, 64), "out": (1, 7, 64)})
        assert attention(one) == Status.ERR_NO_DEVICE
        assert attention(attention_desc(kv_tokens=0), k=None, v=None) == Status.ERR_NO_DEVICE
    code = ctypes.c_int32(0)
    assert lib.dcnv2_cross_attention_read_error(ctypes.byref(d), None, None,
                                                ctypes.byref(code)) == bad
    assert lib.dcnv2_cross_attention_read_error(ctypes.byref(few), None, None, None) == bad
    code.value = 5
    assert lib.dcnv2_cross_attention_read_error(ctypes.byref(few), None, None,
                                                ctypes.byref(code)) == Status.OK
    assert code.value == 0


def test_rotary_tables():
    freqs, axis = rotary_axes(16, [2, 3, 3], base=100.0, device="cpu")
    assert list(axis) == [0, 0, 1, 1, 1, 2, 2, 2]
    assert torch.equal(freqs, torch.tensor([1, 100 ** -0.5, 1, 100 ** (-1 / 3), 100 ** (-2 / 3),
                                            1, 100 ** (-1 / 3), 100 ** (-2 / 3)],
                                           dtype=torch.float32))
    freqs, axis = rotary_axes(16, [4, 2, 2], turns=True, shared_table=True, device="cpu")
    assert list(axis) == [0, 1, 2, 0, 1, 2, 0, 0]
    want = torch.tensor([10000.0 ** (-p / 8) for p in range(8)], dtype=torch.float32)
    assert torch.equal(freqs, want)
    for rot, sections in ((16, [4, 5]), (15, [7]), (0, []), (10, [1] * 5), (4, [3, -1])):
        with pytest.raises(ValueError):
            rotary_axes(rot, sections, device="cpu")


def test_level_positions():
    p = level_positions([(2, 3), (1, 2)], device="cpu")
    assert p.dtype == torch.int32 and p.tolist() == [[
        [0, 0, 0], [0, 0, 1], [0, 0, 2], [0, 1, 0], [0, 1, 1], [0, 1, 2], [1, 0, 0], [1, 0, 1]]]
    with pytest.raises(ValueError):
        level_positions([], device="cpu")
