"""The token operators (dcnv2_qk_norm_rotary, dcnv2_cross_attention) against plain fp64 restatements
of their formulas, and a run of them together behind the levels of a detector step.

Tolerances, from the arithmetic (u = half a step of the output type, e = 2^-24):
  norm, rotation  y = x * r * w: r within 4 roundings and the sum's D/2 * e at most (the products are
                  positive), so y within (D/2 + 8) e; cosine and sine within 2^-21 (fraction of a
                  turn rounded to fp32, sincospif); out = y0 c - y1 s in two roundings, then u:
                  |d| <= u |ref| + (|y0| + |y1|) ((D/2 + 12) e + 2^-21) + the least subnormal / 2
  attention       a score's error is ds = D 2^-23 sum|q k| scale (fp32 accumulation, truncating) +
                  4 e |s| (scale, base-2 exponent); p is off by ds + 2^-21 relatively and by u when
                  rounded for the product with v (fp16: by at least 2^-25 of the largest p); the sums
                  over n states by n 2^-23. With A = sum p|v| / sum p:
                  |d| <= u |ref| + A (u + 2 (ds + 2^-21 + n 2^-23)) + 2^-25 sum|v| / sum p (fp16)
                  lse: ds + 2^-21 + n 2^-23 + 4 e |lse|
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from dcnv2_b200 import (DCNv2Error, capi, dcnv2_cross_attention, dcnv2_forward,  # noqa: E402
                        dcnv2_qk_norm_rotary, level_positions, rotary_axes)
from dcnv2_b200 import workloads as wl  # noqa: E402

DEV = "cuda:0"
E = 2.0 ** -24
FP16, BF16, FP32 = torch.float16, torch.bfloat16, torch.float32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---------------------------------------------------------------- norm and rotation


def plain_rotary(x, pos, freqs, axis, weight, norm, eps, interleaved):
    """fp64 (out, |y0| + |y1| of each element's pair)."""
    x = x.double()
    if norm:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
        if weight is not None:
            x = x * weight.double()
    out, mag = x.clone(), x.abs()
    for p, a in enumerate(axis):
        e0, e1 = (2 * p, 2 * p + 1) if interleaved else (p, p + len(axis))
        ang = (pos[..., a].double() * freqs[p].double())[:, :, None]
        out[..., e0] = x[..., e0] * ang.cos() - x[..., e1] * ang.sin()
        out[..., e1] = x[..., e1] * ang.cos() + x[..., e0] * ang.sin()
        mag[..., e0] = mag[..., e1] = x[..., e0].abs() + x[..., e1].abs()
    return out, mag


def check_rotary(got, x, pos, freqs, axis, weight, norm, eps, interleaved):
    ref, mag = plain_rotary(x, pos, freqs, axis, weight, norm, eps, interleaved)
    tol = half_step(x.dtype) * ref.abs() + \
        mag * ((x.shape[-1] / 2 + 12) * E + 2.0 ** -21) + torch.finfo(x.dtype).smallest_normal * \
        torch.finfo(x.dtype).eps / 2
    err = (got.cpu().double() - ref).abs()
    assert got.dtype == x.dtype and got.shape == x.shape
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("dtype", [FP32, FP16, BF16])
@pytest.mark.parametrize("b,t,hq,hk,d,rot,axes,norm,inter,turns", [
    (1, 1, 1, 0, 2, 2, 1, "rms", False, False),        # one pair
    (2, 1, 32, 8, 128, 128, 1, "rms", False, False),   # single tokens, grouped heads
    (3, 37, 5, 3, 64, 32, 2, "rms", False, False),     # half of the head rotated
    (1, 1021, 0, 4, 80, 80, 3, None, True, True),      # keys only, neighbouring pairs, axes in turn
    (2, 85, 3, 3, 72, 72, 3, "rms", False, True),      # 36 pairs: 8-byte accesses
    (2, 9, 2, 7, 16, 6, 3, "rms", False, False),       # 3 pairs and 10 elements behind: single ones
    (2, 9, 2, 7, 18, 6, 3, "rms", True, False),
    (4, 50, 7, 1, 256, 256, 4, "rms", False, True),    # widest head, four axes
    (4, 50, 7, 1, 254, 126, 4, "rms", False, True),    # scalar path, several chunks per lane
    (1, 3, 300, 300, 256, 256, 1, "rms", True, False),  # a token's heads exceed a block
    (2, 33, 4, 4, 96, 0, 1, "rms", False, False),      # norm alone
    (40, 700, 8, 8, 32, 32, 2, None, False, False),    # many blocks
])
def test_norm_rotary_matches_formula(dtype, b, t, hq, hk, d, rot, axes, norm, inter, turns):
    g = gen(b * 1000 + t + d)
    pairs = rot // 2
    q = (torch.randn(b, t, hq, d, generator=g) * 2).to(dtype) if hq else None
    k = (torch.randn(b, t, hk, d, generator=g) * 2).to(dtype) if hk else None
    qw = (1 + 0.3 * torch.randn(d, generator=g)).to(dtype) if norm and hq else None
    kw = (1 + 0.3 * torch.randn(d, generator=g)).to(dtype) if norm and hk and b > 1 else None
    pos = torch.randint(-5000, 200000, (1 if b == 3 else b, t, axes), generator=g,
                        dtype=torch.int32)
    kwargs = {}
    freqs, axis = None, b""
    if rot:
        sections = [pairs // axes + (i < pairs % axes) for i in range(axes)]
        freqs, axis = rotary_axes(rot, sections, turns=turns, shared_table=turns, device="cpu")
        kwargs = dict(positions=pos.to(DEV), freqs=freqs.to(DEV), pair_axis=axis)
    mv = lambda x: None if x is None else x.to(DEV)  # noqa: E731
    qo, ko = dcnv2_qk_norm_rotary(mv(q), mv(k), q_weight=mv(qw), k_weight=mv(kw), norm=norm,
                                  eps=1e-5, interleaved=inter, **kwargs)
    for got, x, w in ((qo, q, qw), (ko, k, kw)):
        if x is None:
            assert got is None
        else:
            check_rotary(got, x, pos, freqs, axis, w, norm, 1e-5, inter)


def test_norm_rotary_strided_in_place_and_unaligned():
    """Queries and keys as views of one projection, written back in place (neighbours untouched);
    then the same values at an address that allows no vector access: the same bits."""
    g = gen(1)
    b, t, h, d = 2, 19, 3, 64
    proj = torch.randn(b, t, 3, h, d, generator=g).to(BF16)
    freqs, axis = rotary_axes(d, [16, 16], device=DEV)
    pos = level_positions([(19, 1)], DEV)[..., 1:].contiguous()
    w = torch.ones(d, dtype=BF16, device=DEV)
    on = proj.to(DEV)
    args = (pos, freqs, axis)
    q, k = dcnv2_qk_norm_rotary(on[:, :, 0], on[:, :, 1], *args, q_weight=w, norm="rms")
    assert torch.equal(on.cpu(), proj)
    check_rotary(q, proj[:, :, 0], pos.cpu(), freqs.cpu(), axis, None, "rms", 1e-6, False)
    qi, ki = dcnv2_qk_norm_rotary(on[:, :, 0], on[:, :, 1], *args, q_weight=w, norm="rms",
                                  q_out=on[:, :, 0], k_out=on[:, :, 1])
    assert torch.equal(on[:, :, 0], q) and torch.equal(on[:, :, 1], k)
    assert torch.equal(on[:, :, 2].cpu(), proj[:, :, 2])
    odd = torch.empty(b * t * h * d + 1, dtype=BF16, device=DEV)[1:].view(b, t, h, d)
    odd.copy_(proj[:, :, 0])
    out = torch.empty(b, h, t, d, dtype=BF16, device=DEV).transpose(1, 2)  # heads first
    q2, none = dcnv2_qk_norm_rotary(odd, None, *args, q_weight=w, norm="rms", q_out=out)
    assert q2 is out and none is None and torch.equal(out, q)


def test_norm_rotary_far_positions_and_zero_rows():
    """Positions to the ends of int32 keep their angle; all-zero heads stay zero under the norm."""
    d = 64
    freqs, axis = rotary_axes(d, [32], device=DEV)
    pos = torch.tensor([[[2 ** 31 - 1], [-2 ** 31], [0], [123456789]]], dtype=torch.int32)
    x = torch.randn(1, 4, 2, d, generator=gen(2))
    x[0, 2, 1] = 0
    for norm in (None, "rms"):
        y, _ = dcnv2_qk_norm_rotary(x.to(DEV), None, pos.to(DEV), freqs, axis, norm=norm)
        check_rotary(y, x, pos, freqs.cpu(), axis, None, norm, 1e-6, False)
        assert not bool(y[0, 2, 1].any())


def test_norm_rotary_large_offsets():
    """Rows behind 2^31 elements: a token stride of 2^27 elements over 20 tokens."""
    d, t, step = 32, 20, 2 ** 27
    big = torch.zeros((t - 1) * step + d, dtype=FP16, device=DEV)
    x = big.as_strided((1, t, 1, d), (0, step, d, 1))
    src = torch.randn(1, t, 1, d, generator=gen(3)).half()
    x.copy_(src)
    freqs, axis = rotary_axes(d, [16], device=DEV)
    pos = torch.arange(t, dtype=torch.int32).view(1, t, 1)
    y, _ = dcnv2_qk_norm_rotary(x, None, pos.to(DEV), freqs, axis, norm="rms", q_out=x)
    check_rotary(x, src, pos, freqs.cpu(), axis, None, "rms", 1e-6, False)


# ---------------------------------------------------------------- attention


def plain_attention(q, k, v, lens=None, mask=None, scale=None):
    """fp64 (out, lse, tolerance of out, tolerance of lse)."""
    B, L, H, D = q.shape
    S, G = k.shape[1], k.shape[2]
    scale = 1 / math.sqrt(D) if scale is None else scale
    u = half_step(q.dtype)
    out = torch.zeros(B, L, H, D, dtype=torch.float64)
    lse = torch.full((B, H, L), -math.inf, dtype=torch.float64)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(B):
        keep = torch.ones(S, dtype=torch.bool)
        if lens is not None:
            keep[max(0, min(S, int(lens[b]))):] = False
        if mask is not None:
            keep &= mask[b if mask.shape[0] > 1 else 0].bool()
        n = int(keep.sum())
        if n == 0:
            continue
        for h in range(H):
            kk, vv = k[b, keep, h // (H // G)].double(), v[b, keep, h // (H // G)].double()
            qq = q[b, :, h].double()
            s = qq @ kk.T * scale
            ds = (qq.abs() @ kk.abs().T * scale).amax(1) * D * 2.0 ** -23 + \
                4 * E * s.abs().amax(1)
            p = torch.exp(s - s.amax(1, keepdim=True))
            tot = p.sum(1, keepdim=True)
            out[b, :, h] = p @ vv / tot
            lse[b, h] = torch.logsumexp(s, 1)
            rel = (ds + 2.0 ** -21 + n * 2.0 ** -23)
            tol[b, :, h] = u * out[b, :, h].abs() + (p @ vv.abs() / tot) * (u + 2 * rel)[:, None]
            if q.dtype == FP16:
                tol[b, :, h] += 2.0 ** -25 * (vv.abs().sum(0)[None] / tot + 1)
            tol_lse[b, h] = rel + 4 * E * lse[b, h].abs()
    return out, lse, tol, tol_lse


def check_attention(got, lse, q, k, v, lens=None, mask=None, scale=None):
    ref, ref_lse, tol, tol_lse = plain_attention(q, k, v, lens, mask, scale)
    got, lse = got.cpu().double(), lse.cpu().double()
    assert bool(torch.isfinite(got).all())
    err = (got - ref).abs()
    assert bool((err <= tol).all()), (float((err / tol.clamp_min(1e-300)).max()), float(err.max()))
    empty = torch.isinf(ref_lse)
    assert torch.equal(torch.isinf(lse), empty) and bool((lse[empty] < 0).all())
    d = (lse - ref_lse).abs()[~empty]
    assert bool((d <= tol_lse[~empty]).all()), float((d / tol_lse[~empty]).max())


def attention_inputs(b, L, s, h, g, d, dtype, seed, spread=1.0):
    r = gen(seed)
    q = (torch.randn(b, L, h, d, generator=r) * spread).to(dtype)
    k, v = (torch.randn(b, s, g, d, generator=r).to(dtype) for _ in range(2))
    return q, k, v


def attention_desc(q, k, v, out=None, scale=None):
    B, L, H, D = q.shape
    d = capi.AttentionDesc(B, L, k.shape[1], H, k.shape[2], D,
                           int(capi.DType.BF16 if q.dtype == BF16 else capi.DType.HALF),
                           scale or D ** -0.5)
    for field, t in ((d.q_stride, q), (d.k_stride, k), (d.v_stride, v),
                     (d.out_stride, q if out is None else out)):
        field[:] = t.stride()[:3]
    return d


def run_attention(q, k, v, lens=None, mask=None, **kw):
    """(out, lse) on the GPU, its error words read clear afterwards."""
    mv = lambda x: None if x is None else x.to(DEV)  # noqa: E731
    q, k, v = mv(q), mv(k), mv(v)
    desc = attention_desc(q.contiguous(), k, v)
    ws = torch.full((max(1, capi.attention_workspace_size(desc)),), 255, dtype=torch.uint8,
                    device=DEV)
    res = dcnv2_cross_attention(q, k, v, kv_lens=mv(lens), key_mask=mv(mask), return_lse=True,
                                workspace=ws, **kw)
    st = torch.cuda.current_stream().cuda_stream
    assert capi.cross_attention_error(desc, ws.data_ptr(), st) == 0
    return res


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("b,L,s,h,g,d", [
    (1, 1, 1, 1, 1, 8),            # the smallest
    (1, 1, 127, 8, 8, 64),
    (1, 1, 129, 32, 8, 128),       # single token, grouped heads
    (2, 1, 5456, 8, 8, 32),        # the levels of a detector step
    (1, 1, 20011, 16, 1, 128),     # one kv head, a long axis
    (2, 3, 300, 64, 2, 72),        # 96 rows per kv head
    (3, 17, 1000, 4, 4, 40),
    (1, 128, 128, 2, 2, 128),      # exact tiles
    (1, 129, 257, 2, 2, 128),      # one more
    (2, 197, 1021, 6, 2, 80),      # odd, grouped: 591 rows per kv head
    (1, 300, 77, 8, 8, 64),        # short states
    (1, 1000, 700, 3, 3, 96),
    (2, 256, 384, 2, 1, 16),
    (1, 513, 130, 2, 2, 104),
    (1, 2, 300, 256, 1, 64),       # a group of more rows than a tile, cut in two
    (1, 3, 200, 131, 1, 64),       # a prime group of more than 128 heads
    (1, 40, 260, 7, 1, 128),       # 18 tokens of 7 heads in a tile
    (21, 300, 200, 4, 4, 64),      # more items than SMs: no split, several items per CTA
    (20, 290, 150, 4, 4, 128),
    (90, 20, 140, 2, 2, 32),       # one tile of rows, more items than SMs
])
def test_attention_matches_formula(dtype, b, L, s, h, g, d):
    q, k, v = attention_inputs(b, L, s, h, g, d, dtype, b + L + s)
    out, lse = run_attention(q, k, v)
    check_attention(out, lse, q, k, v)


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("L,h,g,d", [(1, 8, 8, 64), (1, 16, 2, 128), (150, 4, 4, 32),
                                     (300, 4, 2, 128)])
def test_attention_lengths_and_masks(dtype, L, h, g, d):
    """Lengths of none, one, tile ends, beyond the states and below zero; masks that leave a
    sequence empty, one state, whole tiles out, the last state only; both together."""
    s = 700
    lens = torch.tensor([0, 1, 127, 128, 129, 700, 9999, -5], dtype=torch.int32)
    b = len(lens)
    q, k, v = attention_inputs(b, L, s, h, g, d, dtype, L + d)
    out, lse = run_attention(q, k, v, lens)
    check_attention(out, lse, q, k, v, lens)
    mask = torch.rand(b, s, generator=gen(5)) < 0.6
    mask[0] = False
    mask[1] = False
    mask[1, 613] = True
    mask[2, 100:600] = False      # whole tiles left out
    mask[3] = False
    mask[3, -1] = True
    mask[4, :256] = False
    mask[5, 64:] = False
    out, lse = run_attention(q, k, v, mask=mask)
    check_attention(out, lse, q, k, v, mask=mask)
    out, lse = run_attention(q, k, v, lens, mask.to(torch.uint8) * 255)
    check_attention(out, lse, q, k, v, lens, mask)
    out, lse = run_attention(q, k, v, lens, mask[2:3])  # one mask for all sequences
    check_attention(out, lse, q, k, v, lens, mask[2:3])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("by_mask", [False, True])
def test_attention_runs_of_empty_sequences(d, by_mask):
    """Several items per CTA, most sequences of the batch without a kept state, in long runs: by
    their length or by their mask; the last and the first one too."""
    b, L, s, h = 64, 260, 300, 2
    q, k, v = attention_inputs(b, L, s, h, h, d, BF16, d)
    lens = torch.zeros(b, dtype=torch.int32)
    lens[[7, 8, 40, 50]] = torch.tensor([300, 1, 129, 128], dtype=torch.int32)
    mask = torch.arange(s) < lens[:, None]
    out, lse = run_attention(q, k, v, **({"mask": mask} if by_mask else {"lens": lens}))
    some = [0, 7, 8, 39, 40, 41, 50, 63]
    check_attention(out[some], lse[some], q[some], k[some], v[some], lens[some])
    gone = (lens == 0).nonzero()[:, 0].to(DEV)
    assert not bool(out[gone].any()) and bool((lse[gone] == -math.inf).all())


@pytest.mark.parametrize("L,h,g,d", [(150, 2, 2, 40), (300, 2, 2, 128), (20, 4, 2, 64)])
def test_attention_long_masked_runs(L, h, g, d):
    """Kept states far apart, at every place of a run of mask words, lengths that end in a run."""
    s = 2611
    mask = torch.zeros(6, s, dtype=torch.bool)
    mask[0, ::257] = True
    mask[1, 63::64] = True
    mask[2, 1023] = mask[2, 1024] = mask[2, -1] = True
    mask[3, :40] = mask[3, 900:1300] = True
    mask[4, 255:257] = mask[4, 2304:] = True
    lens = torch.tensor([2611, 2000, 2610, 1200, 2559, 0], dtype=torch.int32)
    q, k, v = attention_inputs(6, L, s, h, g, d, BF16, L + d + 1)
    out, lse = run_attention(q, k, v, mask=mask)
    check_attention(out, lse, q, k, v, mask=mask)
    out, lse = run_attention(q, k, v, lens, mask)
    check_attention(out, lse, q, k, v, lens, mask)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, -65504.0])
@pytest.mark.parametrize("L,h,g,d", [(1, 8, 2, 64), (200, 2, 2, 128)])
def test_attention_unkept_states_reach_nothing(L, h, g, d, bad):
    """States that lengths or mask leave out hold NaN, infinities, the type's lowest value: the
    result has the bits it has with zeros there."""
    s = 523
    lens = torch.tensor([300, 523, 0], dtype=torch.int32)
    mask = torch.rand(3, s, generator=gen(6)) < 0.7
    mask[1, 128:256] = False
    q, k, v = attention_inputs(3, L, s, h, g, d, FP16, 7)
    gone = ~mask | (torch.arange(s) >= lens[:, None])
    clean = [torch.where(gone[:, :, None, None], torch.zeros((), dtype=FP16), x) for x in (k, v)]
    dirty = [torch.where(gone[:, :, None, None], torch.full((), bad, dtype=FP16), x)
             for x in (k, v)]
    want = run_attention(q, *clean, lens, mask)
    got = run_attention(q, *dirty, lens, mask)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    check_attention(*got, q, *clean, lens, mask)


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("L", [1, 140])
def test_attention_steep_scores(dtype, L):
    """Scores that rise, fall or peak along the states by hundreds: the running maximum moves in
    every tile, and nothing overflows or is lost."""
    s, d = 1200, 64
    q = torch.ones(3, L, 2, d).to(dtype)
    ramp = torch.linspace(-3, 3, s)
    k = torch.stack([ramp, -ramp, 3 - 6 * ((torch.arange(s) - 700).abs() / 700.0)])
    k = k[:, :, None, None].expand(3, s, 2, d).contiguous().to(dtype)
    v = torch.randn(3, s, 2, d, generator=gen(8)).to(dtype)
    for scale in (None, 2.0, 1e-4):
        out, lse = run_attention(q, k, v, scale=scale)
        check_attention(out, lse, q, k, v, scale=scale)


def test_attention_strides_layouts_and_shared_states():
    """Fused projections, caches laid out heads first, shared (expanded) states and heads, outputs in
    a wider buffer whose other places stay as they are, no lse: the bits of the contiguous call."""
    b, L, s, h, g, d = 3, 70, 333, 4, 2, 64
    q, k, v = (x.to(DEV) for x in attention_inputs(b, L, s, h, g, d, BF16, 9))
    want, lse = dcnv2_cross_attention(q, k, v, return_lse=True)
    kv = torch.stack([k, v], 2)
    assert torch.equal(dcnv2_cross_attention(q, kv[:, :, 0], kv[:, :, 1]), want)
    kh, vh = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    qh = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(dcnv2_cross_attention(qh, kh, vh), want)
    wide = torch.full((b, L, h + 1, d + 8), 7.0, dtype=BF16, device=DEV)
    assert torch.equal(dcnv2_cross_attention(q, k, v, out=wide[:, :, 1:, :d]), want)
    assert bool((wide[:, :, 0] == 7).all()) and bool((wide[..., d:] == 7).all())
    ke, ve = (x[:1].expand(b, s, g, d) for x in (k, v))
    assert torch.equal(dcnv2_cross_attention(q, ke, ve),
                       dcnv2_cross_attention(q, ke.contiguous(), ve.contiguous()))
    k1, v1 = (x[:, :, :1].expand(b, s, g, d) for x in (k, v))
    assert torch.equal(dcnv2_cross_attention(q, k1, v1),
                       dcnv2_cross_attention(q, k1.contiguous(), v1.contiguous()))
    # one query repeated over the batch
    qe = q[:1].expand(b, L, h, d)
    assert torch.equal(dcnv2_cross_attention(qe, k, v), dcnv2_cross_attention(qe.contiguous(), k, v))


@pytest.mark.parametrize("d", [40, 64, 72, 128])
def test_attention_outputs_beside_others(d):
    """Outputs as a view of a wider buffer, with more items than SMs (whole tiles of rows leave at
    once): the places around them stay as they were."""
    b, L, s, h = 30, 273, 90, 3
    q, k, v = (x.to(DEV) for x in attention_inputs(b, L, s, h, h, d, FP16, d))
    want = dcnv2_cross_attention(q, k, v)
    wide = torch.full((b, L + 2, h + 1, 136), 7.0, dtype=FP16, device=DEV)
    got = dcnv2_cross_attention(q, k, v, out=wide[:, 1:-1, 1:, :d])
    assert torch.equal(got, want)
    wide[:, 1:-1, 1:, :d] = 7
    assert bool((wide == 7).all())
    check_attention(want[:2], dcnv2_cross_attention(q, k, v, return_lse=True)[1][:2],
                    q[:2].cpu(), k[:2].cpu(), v[:2].cpu())


def test_attention_shared_query_and_two_streams_at_once():
    """One query for all sequences (batch stride 0) on each kernel; two calls at once on two streams,
    each with a workspace of its own, give the bits they give alone."""
    for L in (1, 30, 200):
        q, k, v = (x.to(DEV) for x in attention_inputs(3, L, 400, 4, 2, 64, BF16, L))
        qe = q[:1].expand(3, L, 4, 64)
        assert torch.equal(dcnv2_cross_attention(qe, k, v),
                           dcnv2_cross_attention(qe.contiguous(), k, v))
    a = [x.to(DEV) for x in attention_inputs(4, 900, 3000, 8, 8, 64, FP16, 1)]
    b = [x.to(DEV) for x in attention_inputs(8, 1, 20000, 16, 2, 128, BF16, 2)]
    want = dcnv2_cross_attention(*a), dcnv2_cross_attention(*b)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, (st, args) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(st):
                got[i].append(dcnv2_cross_attention(*args))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_attention_large_offsets():
    """States behind 2^31 elements: a token stride of 2^23 elements over 300 tokens."""
    s, d, step = 300, 64, 2 ** 23
    big = torch.zeros((s - 1) * step + 2 * d, dtype=FP16, device=DEV)
    k = big.as_strided((1, s, 1, d), (0, step, d, 1))
    v = big[d:].as_strided((1, s, 1, d), (0, step, d, 1))
    for L in (1, 130):
        q, kk, vv = attention_inputs(1, L, s, 1, 1, d, FP16, 10 + L)
        k.copy_(kk)
        v.copy_(vv)
        out, lse = dcnv2_cross_attention(q.to(DEV), k, v, return_lse=True)
        check_attention(out, lse, q, kk, vv)


def test_attention_no_states_and_empty_batches():
    q = torch.randn(2, 3, 4, 64, device=DEV).half()
    k = torch.empty(2, 0, 2, 64, device=DEV, dtype=FP16)
    out, lse = dcnv2_cross_attention(q, k, k, return_lse=True)
    assert not bool(out.any()) and bool((lse == -math.inf).all())
    for shape in ((0, 3, 4, 64), (2, 0, 4, 64)):
        q0 = torch.empty(shape, device=DEV, dtype=FP16)
        k0 = torch.empty(shape[0], 5, 2, 64, device=DEV, dtype=FP16)
        out, lse = dcnv2_cross_attention(q0, k0, k0, return_lse=True)
        assert out.shape == q0.shape and lse.shape == (shape[0], 4, shape[1])
        assert dcnv2_qk_norm_rotary(q0, None, norm="rms")[0].shape == q0.shape


def test_attention_same_bits_every_time_and_error_word_clear():
    q, k, v = (x.to(DEV) for x in attention_inputs(2, 1, 9000, 8, 2, 128, BF16, 11))
    first = dcnv2_cross_attention(q, k, v)
    for _ in range(20):
        assert torch.equal(dcnv2_cross_attention(q, k, v), first)
    q, k, v = (x.to(DEV) for x in attention_inputs(2, 60, 9000, 8, 2, 128, BF16, 12))
    first, lse = run_attention(q, k, v)  # (a workspace that holds anything, read clear)
    for _ in range(20):
        again = run_attention(q, k, v)
        assert torch.equal(again[0], first) and torch.equal(again[1], lse)


def test_refusals_on_the_device():
    """What the wrappers refuse, and alignment that the C call refuses, launches nothing."""
    q = torch.randn(1, 4, 4, 64, device=DEV).half()
    k = torch.randn(1, 9, 2, 64, device=DEV).half()
    ok = dcnv2_cross_attention(q, k, k)
    bad = [
        (ValueError, lambda: dcnv2_cross_attention(q, k[..., :56], k)),
        (ValueError, lambda: dcnv2_cross_attention(q, k, k.cpu())),
        (TypeError, lambda: dcnv2_cross_attention(q, k, k.bfloat16())),
        (TypeError, lambda: dcnv2_cross_attention(q.float(), k.float(), k.float())),
        (ValueError, lambda: dcnv2_cross_attention(q.transpose(2, 3), k, k)),
        (DCNv2Error, lambda: dcnv2_cross_attention(q[:, :, :3], k, k)),
        (DCNv2Error, lambda: dcnv2_cross_attention(q, k, k, scale=-1.0)),
        (DCNv2Error, lambda: dcnv2_cross_attention(q, k, k, scale=math.nan)),
        (DCNv2Error, lambda: dcnv2_cross_attention(q[..., :60], k[..., :60], k[..., :60])),
        (DCNv2Error, lambda: dcnv2_cross_attention(q[..., 4:44], k[..., 4:44], k[..., 4:44])),
        (TypeError, lambda: dcnv2_cross_attention(q, k, k, kv_lens=torch.ones(1, device=DEV))),
        (ValueError, lambda: dcnv2_cross_attention(
            q, k, k, key_mask=torch.ones(1, 8, dtype=torch.bool, device=DEV))),
        (TypeError, lambda: dcnv2_cross_attention(q, k, k, key_mask=torch.ones(1, 9, device=DEV))),
        (ValueError, lambda: dcnv2_cross_attention(q, k, k, out=q[:, :3])),
        (ValueError, lambda: dcnv2_cross_attention(
            q, k, k, workspace=torch.empty(1, dtype=torch.uint8, device=DEV).expand(4096))),
        (DCNv2Error, lambda: dcnv2_cross_attention(
            q, k, k, out=torch.empty(4096, dtype=FP16, device=DEV).as_strided(
                q.shape, (1024, 64, 64, 1)))),
        (ValueError, lambda: dcnv2_qk_norm_rotary(None, None)),
        (TypeError, lambda: dcnv2_qk_norm_rotary(q.double(), None, norm="rms")),
        (ValueError, lambda: dcnv2_qk_norm_rotary(q, k, norm="rms")),
        (ValueError, lambda: dcnv2_qk_norm_rotary(q, None, norm="layer")),
        (ValueError, lambda: dcnv2_qk_norm_rotary(q, None, q_weight=q[0, 0, 0])),
        (ValueError, lambda: dcnv2_qk_norm_rotary(q, None, freqs=torch.ones(2, device=DEV),
                                                  pair_axis=b"\0\0")),
        (DCNv2Error, lambda: dcnv2_qk_norm_rotary(
            q, None, torch.zeros(1, 4, 1, dtype=torch.int32, device=DEV),
            torch.ones(2, device=DEV), b"\0\1")),
        (DCNv2Error, lambda: dcnv2_qk_norm_rotary(q[..., :63], None, norm="rms")),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()
    assert torch.equal(dcnv2_cross_attention(q, k, k), ok)


# ---------------------------------------------------------------- together


def _decoder_step(dev=DEV):
    """Tensors of a decoder step behind the levels: DCNv2 maps -> tokens -> normed, rotated keys and
    values; queries normed, rotated, attending under the padding mask."""
    g = gen(12)
    sizes, c, heads, B, L = [(16, 16), (8, 8), (4, 4)], 64, 4, 2, 19
    maps = []
    for i, (h, w) in enumerate(sizes):
        inp = wl.make_layer_inputs(wl.Layer(B, c, h, w, c), "fp16", 0.1, 3.0, 0.5, seed=i).to(dev)
        maps.append(dcnv2_forward(*inp.tensors()))
    tokens = torch.cat([m.flatten(2).transpose(1, 2) for m in maps], 1)
    wkv = (torch.randn(c, 2 * c, generator=g) / c ** 0.5).half().to(dev)
    S = tokens.shape[1]
    kv = (tokens.reshape(-1, c) @ wkv).view(B, S, 2, heads, c // heads)
    q = torch.randn(B, L, heads, c // heads, generator=g).half().to(dev)
    gain = (1 + 0.1 * torch.randn(c // heads, generator=g)).half().to(dev)
    pos = level_positions(sizes, dev)
    qpos = torch.randint(0, 16, (B, L, 3), generator=g, dtype=torch.int32).to(dev)
    freqs, axis = rotary_axes(c // heads, [2, 3, 3], base=100.0, device=dev)
    mask = torch.cat([((torch.arange(h) < h * 3 // 4)[:, None] &
                       (torch.arange(w) < w // 2)[None]).flatten() for h, w in sizes])
    mask = torch.stack([mask, torch.ones_like(mask)]).to(dev)
    return dict(q=q, kv=kv, pos=pos, qpos=qpos, freqs=freqs, axis=axis, gain=gain, mask=mask)


def _decode(t, ws=None):
    q, _ = dcnv2_qk_norm_rotary(t["q"], None, t["qpos"], t["freqs"], t["axis"],
                                q_weight=t["gain"], norm="rms")
    _, k = dcnv2_qk_norm_rotary(None, t["kv"][:, :, 0], t["pos"], t["freqs"], t["axis"],
                                k_weight=t["gain"], norm="rms")
    return dcnv2_cross_attention(q, k, t["kv"][:, :, 1], key_mask=t["mask"], return_lse=True,
                                 workspace=ws) + (q, k)


def test_levels_tokens_rotation_and_attention_together():
    t = _decoder_step()
    out, lse, q, k = _decode(t)
    cpu = {n: (x.cpu() if torch.is_tensor(x) else x) for n, x in t.items()}
    check_rotary(q, cpu["q"], cpu["qpos"], cpu["freqs"], t["axis"], cpu["gain"], "rms", 1e-6, False)
    check_rotary(k, cpu["kv"][:, :, 0], cpu["pos"], cpu["freqs"], t["axis"], cpu["gain"], "rms",
                 1e-6, False)
    check_attention(out, lse, q.cpu(), k.cpu(), cpu["kv"][:, :, 1], mask=cpu["mask"])


def test_together_on_another_stream_and_in_two_graphs():
    """The same bits on a side stream, through raw stream handles, and from two captured graphs that
    are replayed one after the other with new inputs written in place."""
    t = _decoder_step()
    want = _decode(t)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _decode(t)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    q, _ = dcnv2_qk_norm_rotary(t["q"], None, t["qpos"], t["freqs"], t["axis"],
                                q_weight=t["gain"], norm="rms", stream=side.cuda_stream)
    out = dcnv2_cross_attention(q, want[3], t["kv"][:, :, 1], key_mask=t["mask"],
                                stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(out, want[0])
    ws = torch.empty(4096, dtype=torch.uint8, device=DEV)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = _decode(t, ws)
        graphs.append((g, res))
    keep = t["q"].clone()
    for scale in (1.0, 3.0, 1.0):
        t["q"].copy_(keep * scale)
        for g, res in graphs:
            g.replay()
        want = _decode(t)
        torch.cuda.synchronize()
        for _, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(res, want))
