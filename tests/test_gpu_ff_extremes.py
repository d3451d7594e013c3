"""Activations and slopes where g is huge but finite: no intermediate overflow may turn a
finite result into a NaN.  Identity matrices pass g and the slope through exactly (or, in
f32's split modes, to 2^-20)."""
from __future__ import annotations

import pytest
import torch

from zengpu_b200 import Activation, GemmMode, kernels as K

pytestmark = pytest.mark.gpu

VALUES = {torch.float32: (1e5, 1e13, 1e19, 3e19, 1e25, 1e38, 3e38), torch.float16: (1e3, 65504.0),
          torch.bfloat16: (1e5, 1e13, 1e19, 3e19, 1e25, 1e38, 3e38)}


@pytest.mark.parametrize("act", list(Activation), ids=lambda a: a.name)
@pytest.mark.parametrize("n", [16, 80], ids=["few_rows", "many_rows"])
@pytest.mark.parametrize("kind", list(VALUES), ids=lambda k: str(k).split(".")[1])
@pytest.mark.parametrize("mode", [GemmMode.TF32X3, GemmMode.SIMT_FP32], ids=lambda m: m.name)
def test_huge_g(mode, kind, n, act):
    eye = torch.eye(n, device="cuda").to(kind)
    one = torch.ones(n, n, device="cuda").to(kind)
    for value in VALUES[kind]:
        for sign in (1.0, -1.0):
            g = (one.float() * (sign * value)).to(kind)
            y, saved = K.gated_ff(eye, g, one, eye, act=act, mode=mode, save=True)
            _, dwg, dwu, _ = K.gated_ff_backward(one, eye, g, one, eye, saved, act=act, mode=mode)
            # every activation is g or 0 there, its slope 1 or 0
            for name, got, want in (("act", y, g.double() if sign > 0 else 0 * g.double()),
                                    ("du", dwu, g.double() if sign > 0 else 0 * g.double()),
                                    ("slope", dwg, one.double() * (sign > 0))):
                bad = (got.double() - want).abs() > 2.0 ** -20 * want.abs()
                assert not bad.any() and torch.isfinite(got).all(), (name, sign * value)
