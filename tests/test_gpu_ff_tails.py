"""The activations and their slopes on 16-bit tensors from g = -30 to 30, in relative
terms: through identity matrices every product is exact, so that each result is the
epilogue's f32 value rounded once.

Bounds.  u = eps / 2 for that rounding, and 2^-14 of the value's size for the f32
arithmetic before it: |g| and |q| are at most 87 where a result is above the smallest
normal bf16, so rounding the exponential's argument (2^-24 of it for each of three
operations) loses 87 * 3 * 2^-24 = 1.6e-5, and the exponential itself 2 + 1.173 * 87
units, 104 * 2^-23 = 1.3e-5; reciprocals and products are a few units; the polynomial
for erfc may add 2^-16: 4.5e-5 together.  A slope is a sum of two terms, which may
cancel: the size is theirs together.  Below f16's smallest normal number half its
smallest step counts.  In bf16 the factor s or c (1 / (1 + e^-x), by a reciprocal that
takes numbers below f32's smallest normal one, 2^-126, as zero) may lose 2^-126; a result
is that factor times |g|, and a slope's second term is s or c times others, so a result
may lose 2^-126 times its size over the factor."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_gated_ff import act64
from zengpu_b200 import Activation, kernels as K

pytestmark = pytest.mark.gpu

TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}


def slope_terms(g, act):
    """The magnitudes of the slope's first term, s or c, and of its second."""
    if act == Activation.RELU:
        return (g > 0).double(), torch.zeros_like(g)
    value, slope = act64(g, act)
    first = torch.where(g != 0, value / torch.where(g != 0, g, 1.0), 0.5).abs()
    return first, (slope - first).abs()


def check(got, want, size, factor, kind, name):
    lost = TINY[kind] * (torch.where(factor > 0, size / factor, 0.0).clamp_min(1.0)
                         if kind == torch.bfloat16 else 1.0)
    bound = torch.finfo(kind).eps / 2 * want.abs() + 2.0 ** -14 * size + lost
    worst = ((got.double() - want).abs() / bound).flatten()
    assert torch.isfinite(got).all()
    assert float(worst.max()) <= 1.0, (name, float(worst.max()), float(want.flatten()[worst.argmax()]))


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("act", list(Activation), ids=lambda a: a.name)
@pytest.mark.parametrize("m", [64, 128], ids=["few_rows", "pairs"])
def test_tails(m, act, kind):
    k, f = m, 1024
    eye, out = torch.eye(k, device="cuda").to(kind), torch.eye(f, device="cuda").to(kind)
    g = torch.linspace(-30, 30, k * f, device="cuda").view(f, k).t().contiguous().to(kind)
    ones = torch.ones(k, f, device="cuda").to(kind)
    y, saved = K.gated_ff(eye, g, ones, out, act=act, save=True)  # h = act(g)
    assert torch.equal(saved[0], g.float()) and torch.equal(saved[1], ones.float())
    value, slope = act64(g.double(), act)
    first, second = slope_terms(g.double(), act)
    check(y, value, value.abs(), first, kind, "act")
    # dh = 1: dg = slope and du = act(g), summed over the rows of an identity
    _, dwg, dwu, dwd = K.gated_ff_backward(ones, eye, g, ones, out, saved, act=act)
    check(dwg, slope, first + second, first, kind, "slope")
    check(dwu, value, value.abs(), first, kind, "du")
    assert K.kernel_status() == 0
