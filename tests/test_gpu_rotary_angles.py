"""Angles of dcnv2_qk_norm_rotary far out: positions to the ends of int32 and frequencies above one,
against the turns position * freq / 2 pi taken exactly (rationals, 1 / 2 pi to 60 digits).

Tolerance: the angle's fraction of a turn is rounded to fp32, 2^-26 turns or 2^-23.3 radians; sine and
cosine are within 2^-23; products and their sum round three times by 2^-24; 16-bit outputs round once
more, and their hardware sines are within 2^-21.1: below 2^-21 and 2^-20 of |x0| + |x1|, beside half a
step of the output."""
import math
import random
from fractions import Fraction

import pytest
import torch

pytestmark = pytest.mark.gpu

from dcnv2_b200 import dcnv2_qk_norm_rotary  # noqa: E402

DEV = "cuda:0"
INV_2PI = Fraction("0.159154943091895335768883763372514362034459645740456448747667")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("top", [1.0, 40.0, 3e4, -1.0])
def test_far_angles(dtype, top):
    r = random.Random(5)
    pairs = 16
    freqs = torch.tensor([top * r.random() for _ in range(pairs)], dtype=torch.float32)
    places = [2 ** 31 - 1, -2 ** 31, 2 ** 30 + 1, -(2 ** 29) - 7, 123456789, 99991, 1, 0]
    x = torch.randn(1, len(places), 1, 2 * pairs, generator=torch.Generator().manual_seed(3)).to(dtype)
    pos = torch.tensor(places, dtype=torch.int32).view(1, -1, 1)
    y, _ = dcnv2_qk_norm_rotary(x.to(DEV), None, pos.to(DEV), freqs.to(DEV), bytes(pairs))
    y, x = y.cpu().double()[0, :, 0], x.double()[0, :, 0]
    half = torch.finfo(dtype).eps / 2
    for t, place in enumerate(places):
        for p in range(pairs):
            a = 2 * math.pi * float(Fraction(freqs[p].item()) * place * INV_2PI % 1)
            e0, e1 = float(x[t, p]), float(x[t, p + pairs])
            tol = (abs(e0) + abs(e1)) * (2.0 ** -21 if dtype == torch.float32 else 2.0 ** -20)
            for got, want in ((y[t, p], e0 * math.cos(a) - e1 * math.sin(a)),
                              (y[t, p + pairs], e1 * math.cos(a) + e0 * math.sin(a))):
                least = torch.finfo(dtype).smallest_normal * half
                assert abs(float(got) - want) <= tol + half * abs(want) + least, (place, p)
