"""dcnv2_cross_attention, state by state: that each kept state counts once, wherever chunks, tiles,
warps and CTAs meet, and that states which are not kept count nowhere, in every form of the kernel.

All scores are 0 here (zero queries), so that every probability, sum and factor of a join is a power of
two or a whole number, exact in fp32: n kept states give lse = log n and the mean of v. In one call
element d of v is 1024 at one state of its own and 0 elsewhere, and the calls go through all states:
out[d] is 1024 / n where that state is kept, else 0. Tolerances: the quotient and the product round by
2^-24 each, the output by half a step of its type (and half its least step); log2 of n (scaled by up to
2^7, below 2^23) is within 2^-23 of at most 23, and lse within 2^-18, where one state of 20011 makes
2^-14.3."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from dcnv2_b200 import dcnv2_cross_attention  # noqa: E402

DEV = "cuda:0"
FP16, BF16 = torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def each_state(b, L, s, h, g, d, dtype, lens, mask):
    q = torch.zeros(b, L, h, d, dtype=dtype, device=DEV)
    k = torch.randn(b, s, g, d, generator=gen(s), device=DEV).to(dtype)
    keep = torch.ones(b, s, dtype=torch.bool, device=DEV)
    if lens is not None:
        keep &= torch.arange(s, device=DEV) < lens[:, None]
    if mask is not None:
        keep &= mask
    n = keep.sum(1).double()
    want_lse = n.log()[:, None, None].expand(b, h, L)
    half = torch.finfo(dtype).eps / 2
    value = (1024 / n.clamp_min(1))[:, None].expand(b, d)
    for at in range(0, s, d):
        states = torch.arange(at, min(s, at + d), device=DEV)
        v = torch.zeros(b, s, g, d, dtype=dtype, device=DEV)
        v[:, states, :, states - at] = 1024
        out, lse = dcnv2_cross_attention(q, k, v, kv_lens=lens, key_mask=mask, return_lse=True)
        want = torch.zeros(b, d, dtype=torch.float64, device=DEV)
        want[:, :len(states)] = value[:, :len(states)] * keep[:, states]
        want = want[:, None, None].expand(b, L, h, d)
        tol = want * (half + 2.0 ** -22) + torch.finfo(dtype).smallest_normal * half
        bad = (out.double() - want).abs() > tol
        assert not bool(bad.any()), (at, bad.nonzero()[0].tolist())
        some = n > 0
        assert bool(((lse.double() - want_lse)[some].abs() <= 2.0 ** -18).all()), at
        assert bool((lse[~some] == -math.inf).all())


FORMS = [
    (1, 1, 20011, 16, 1, 128, BF16),  # single token, one kv head: 16 CTAs of 4 warps share the states
    (1, 1, 20011, 8, 1, 64, FP16),
    (2, 1, 5456, 8, 8, 32, FP16),     # one CTA or two per head
    (1, 20, 9001, 4, 1, 128, FP16),   # one tile of rows: two warpgroups, a cluster of 8
    (1, 20, 9001, 4, 1, 64, BF16),
    (1, 150, 9001, 1, 1, 128, BF16),  # tiles of rows, split over a cluster
    (1, 530, 9001, 1, 1, 64, FP16),
    (50, 290, 300, 3, 3, 64, BF16),   # items in turn, no split
    (50, 290, 300, 3, 3, 128, FP16),
]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("masked", [False, True])
def test_each_kept_state_counts_once(form, masked):
    b, _, s = form[:3]
    lens = mask = None
    if masked:
        lens = torch.randint(0, s + 1, (b,), generator=gen(1), device=DEV, dtype=torch.int32)
        lens[0] = s - 5
        mask = torch.rand(b, s, generator=gen(2), device=DEV) < 0.7
        mask[:, s // 3:s // 2] = False
    each_state(*form, lens, mask)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, -65504.0])
@pytest.mark.parametrize("b,L,h,g,d", [
    (3, 1, 4, 2, 32),      # single tokens, heads of up to 32
    (3, 20, 4, 2, 64),     # one tile of rows
    (3, 20, 4, 2, 128),
    (3, 530, 2, 2, 64),    # four warpgroups, tiles of 64 states, split
    (80, 130, 2, 2, 64),   # items in turn
    (80, 130, 2, 2, 128),
])
def test_unkept_states_reach_nothing_in_any_form(b, L, h, g, d, bad):
    """States that are left out by length, by single places or by whole tiles hold NaN, infinities, the
    type's lowest value: the bits are those with zeros there."""
    s = 523
    q = torch.randn(b, L, h, d, generator=gen(3), device=DEV).half()
    k, v = (torch.randn(b, s, g, d, generator=gen(i), device=DEV).half() for i in (4, 5))
    lens = torch.full((b,), s, dtype=torch.int32, device=DEV)
    lens[0], lens[1] = 300, 0
    mask = torch.rand(b, s, generator=gen(6), device=DEV) < 0.7
    mask[2, 128:256] = False
    gone = (~mask | (torch.arange(s, device=DEV) >= lens[:, None]))[:, :, None, None]

    def run(fill):
        kk, vv = (torch.where(gone, torch.full((), fill, dtype=FP16, device=DEV), x) for x in (k, v))
        return dcnv2_cross_attention(q, kk, vv, kv_lens=lens, key_mask=mask, return_lse=True)

    want, got = run(0.0), run(bad)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert bool(torch.isfinite(got[0]).all())


@pytest.mark.parametrize("b,L,s,group,g,d", [
    (5, 200, 191, 3, 1, 104), (3, 129, 3000, 33, 1, 96), (9, 300, 700, 7, 2, 64),
    (2, 20, 3000, 5, 2, 128), (2, 20, 3000, 5, 2, 64), (90, 129, 256, 33, 1, 48),
    (60, 290, 700, 3, 2, 128),
])
def test_bits_do_not_depend_on_what_ran_before(b, L, s, group, g, d):
    """Groups of heads that leave rows of a tile unused, between calls that leave other values in an
    SM's shared memory: the same bits every time."""
    h = group * g
    q = torch.randn(b, L, h, d, generator=gen(7), device=DEV).half()
    k, v = (torch.randn(b, s, g, d, generator=gen(i), device=DEV).half() for i in (8, 9))
    full = torch.randn(40, 1024, 8, d, generator=gen(10), device=DEV).half()
    want = dcnv2_cross_attention(q, k, v, return_lse=True)
    for scale in (100.0, -1000.0, 0.0, 30.0, math.nan, math.inf):
        dcnv2_cross_attention(full * scale, full, full)
        got = dcnv2_cross_attention(q, k, v, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("b,L,h,g,d", [(2, 1, 4, 2, 32), (2, 20, 4, 2, 64), (2, 300, 2, 2, 128),
                                       (80, 130, 2, 2, 64)])
def test_infinities_among_kept_states(b, L, h, g, d):
    """Kept scores of -inf count as nothing: a row that has only those gives zeros and lse = -inf, one
    that has others the result without them. NaN among the kept states shows in the rows that read it
    and in no others."""
    s = 300
    q = torch.rand(b, L, h, d, generator=gen(11), device=DEV).half() + 0.5
    k, v = (torch.randn(b, s, g, d, generator=gen(i), device=DEV).half() for i in (12, 13))
    gone = torch.rand(b, s, generator=gen(14), device=DEV) < 0.3
    gone[0] = True
    low = torch.where(gone[:, :, None, None], torch.full((), -math.inf, dtype=FP16, device=DEV), k)
    out, lse = dcnv2_cross_attention(q, low, v, return_lse=True)
    want, want_lse = dcnv2_cross_attention(q, k, v, key_mask=~gone, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    assert not bool(out[0].any()) and bool((lse[0] == -math.inf).all())
    v = v.clone()
    v[-1, 5, 0, 3] = math.nan
    k = k.clone()
    k[1, 299, g - 1, 7] = math.nan
    out = torch.isnan(dcnv2_cross_attention(q, k, v))
    want = torch.zeros_like(out)
    want[-1, :, :h // g, 3] = True
    want[1, :, h - h // g:] = True
    assert torch.equal(out, want)
