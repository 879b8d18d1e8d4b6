"""dcnv2_cross_attention where its bounded waits run out: a mask whose search for kept states takes far
longer than a short limit (dcnv2_diag_set_attention_wait_limit). Every wait of the kernel ends by
itself, so the calls return and the device stays usable."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from dcnv2_b200 import (capi, dcnv2_cross_attention, dcnv2_cross_attention_error,  # noqa: E402
                        dcnv2_cross_attention_workspace_size)

DEV = "cuda:0"
S = 2 ** 25  # states under the mask: a search of tens of milliseconds

# sequences, query tokens, heads, kv heads, head_dim of each form of the kernel
FORMS = [
    (3, 20, 4, 2, 64),     # one tile of rows, states split over a cluster
    (3, 20, 4, 2, 128),
    (2, 300, 2, 2, 64),    # several tiles, split
    (2, 300, 2, 2, 128),
    (74, 130, 4, 4, 64),   # two items per CTA, two of four warpgroups without rows
    (37, 300, 4, 4, 128),  # two items per CTA, the second tile of rows of an item short or missing
]


@pytest.fixture
def limit():
    """Sets the limit of the attention's waits for one test, and restores the default."""
    yield capi.set_attention_wait_limit
    capi.set_attention_wait_limit()


def long_call(form, first_kept, again=0, short=True):
    """A call over S states, few of them kept: the first 64 where first_kept, else none (and of every
    2^21 the first `again`, if any). Sequences of the first half are 64 states long, if `short`. The states lie over one another (each starts 8 elements behind
    the last), so that they take little memory."""
    b, L, h, g, d = form
    r = torch.Generator(DEV).manual_seed(b + L + d)
    mem = torch.randn((S - 1) * 8 + d, generator=r, device=DEV, dtype=torch.float16)
    k = mem.as_strided((b, S, g, d), (0, 8, 0, 1))
    q = torch.randn(b, L, h, d, generator=r, device=DEV, dtype=torch.float16)
    mask = torch.zeros(1, S, dtype=torch.bool, device=DEV)
    mask[0, :64] = first_kept
    if again:
        mask.view(-1, 2 ** 21)[:, :again] = True
    lens = torch.full((b,), S, dtype=torch.int32, device=DEV)
    if short:
        lens[:b // 2] = 64
    desc = capi.AttentionDesc(b, L, S, h, g, d, int(capi.DType.HALF), d ** -0.5)
    for field, t in ((desc.q_stride, q), (desc.k_stride, k), (desc.v_stride, k),
                     (desc.out_stride, q)):
        field[:] = t.stride()[:3]
    ws = torch.empty(capi.attention_workspace_size(desc), dtype=torch.uint8, device=DEV)
    out, lse = torch.empty_like(q).fill_(7), None

    def call():
        nonlocal lse
        _, lse = dcnv2_cross_attention(q, k, k, kv_lens=lens, key_mask=mask, return_lse=True,
                                       out=out, workspace=ws)
        code = capi.cross_attention_error(desc, ws.data_ptr(),
                                          torch.cuda.current_stream().cuda_stream)
        return out, lse, code

    kk = mem.as_strided((64, d), (8, 1)).double()
    s = q.double() @ kk.T * d ** -0.5
    want = torch.softmax(s, -1) @ kk if first_kept else torch.zeros_like(q, dtype=torch.float64)
    want_lse = torch.logsumexp(s, -1).transpose(1, 2) if first_kept else torch.full(
        (b, h, L), -math.inf, dtype=torch.float64, device=DEV)
    return call, want, want_lse


def right(out, lse, want, want_lse):
    """[b, h, L]: rows that hold the result. Half a step of the output and of the probabilities (2^-11
    each, of values below 8; 64 states of at most 128 elements: the rest is below 2^-12)."""
    tol = 8 * (2 * 2.0 ** -11 + 2.0 ** -12)
    close = ((out.double() - want).abs() <= tol).all(-1).transpose(1, 2)
    same = (lse.double() - want_lse).abs() <= 1e-3
    return close & (same | (lse.double() == want_lse))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("first_kept", [True, False])
def test_calls_return_and_say_so_when_waits_run_out(limit, form, first_kept):
    """With a limit of 1 ms the error words are set, and with the default one the same call, made
    behind it, is right: no warp waits for one that has given up."""
    call, want, want_lse = long_call(form, first_kept)
    limit(1000)
    assert call()[2] != 0
    limit()
    out, lse, code = call()
    assert code == 0
    assert bool(right(out, lse, want, want_lse).all())


@pytest.mark.parametrize("form", FORMS)
def test_copies_in_flight_are_waited_for_once(limit, form):
    """The issuers give up while a gap of the mask is searched; behind it the producer finds tiles again
    and fills its buffers until a place of V stays taken, with K of that tile on its way. What is in
    flight then lands long before the limit for that, which would take 2 s and show in the error
    words."""
    call, _, _ = long_call(form, True, again=4096)
    call()
    limit(100)
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    code = call()[2]
    end.record()
    end.synchronize()
    assert code and not code & 16
    assert begin.elapsed_time(end) < 1500


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("first_kept,again", [(True, 0), (False, 0), (True, 4096)])
def test_rows_whose_waits_ran_out_are_nan(limit, form, first_kept, again):
    """No row looks like a result that it is not: not like that of a sequence without kept states, not
    like one over a part of the states, and none is left as it was. Rows and their lse are right, or
    NaN from end to end, and those of the sequences that were searched are NaN."""
    call, want, want_lse = long_call(form, first_kept, again)
    limit(100)
    out, lse, code = call()
    assert code
    nan = torch.isnan(out).all(-1).transpose(1, 2) & torch.isnan(lse)
    b = out.shape[0]
    assert bool(nan[b // 2:].all())
    if first_kept:
        assert bool((nan | right(out, lse, want, want_lse))[:b // 2].all())
    else:
        zero = ~out.any(-1).transpose(1, 2) & (lse == -math.inf)
        assert bool((nan | zero)[:b // 2].all())


@pytest.mark.parametrize("d,L", [(64, 130), (128, 130)])
@pytest.mark.parametrize("first_kept", [True, False])
def test_searches_in_a_row_do_not_add_up(limit, d, L, first_kept):
    """Four items per CTA, each with a search of 2^25 states (about 50 ms): a limit that is above the
    time of 2^24 of them and far below that of all does not run out, whoever waits meanwhile."""
    call, want, want_lse = long_call((148, L, 4, 4, d), first_kept, short=False)
    limit(80000)
    out, lse, code = call()
    assert code == 0
    assert bool(right(out, lse, want, want_lse).all())


@pytest.mark.parametrize("L,h,g,d", [(20, 4, 2, 64), (300, 2, 2, 128)])
def test_error_words_through_the_package(limit, L, h, g, d):
    """A caller that keeps the workspace reads the error of its last call, on the stream it ran on, and
    cannot take another tensor for it."""
    q = torch.randn(1, L, h, d, device=DEV).half()
    mem = torch.zeros((S - 1) * 8 + d, device=DEV, dtype=torch.float16)
    k = mem.as_strided((1, S, g, d), (0, 8, 0, 1))
    mask = torch.zeros(1, S, dtype=torch.bool, device=DEV)
    size = dcnv2_cross_attention_workspace_size(q, k, k)
    ws = torch.full((size,), 255, dtype=torch.uint8, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    assert size > 0
    limit(100)
    out = dcnv2_cross_attention(q, k, k, key_mask=mask, workspace=ws, stream=side.cuda_stream)
    assert dcnv2_cross_attention_error(q, k, k, ws, stream=side.cuda_stream) != 0
    assert bool(torch.isnan(out).all())
    limit()
    out = dcnv2_cross_attention(q, k, k, key_mask=mask, workspace=ws)
    assert dcnv2_cross_attention_error(q, k, k, ws) == 0 and not bool(out.any())
    for bad in (None, ws[1:], ws.cpu(), torch.empty(1, dtype=torch.uint8, device=DEV).expand(size)):
        with pytest.raises(ValueError):
            dcnv2_cross_attention_error(q, k, k, bad)
    one = q[:, :1]
    assert dcnv2_cross_attention_workspace_size(one, k, k) == 0
    assert dcnv2_cross_attention_error(one, k, k, None) == 0
