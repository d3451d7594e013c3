"""The gated block's scratch memory holds whatever was there before: a pass gives the
same bits over a workspace of zeros and over one whose every word is a NaN (0xFF bytes),
which a product with a zero does not hide."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_gated_ff import TYPES, inputs
from zengpu_b200 import Activation, GemmMode, kernels as K

pytestmark = pytest.mark.gpu


def all_bits(args, mode):
    x, wg, wu, wd, dy = args
    y, saved = K.gated_ff(x, wg, wu, wd, act=Activation.SILU, mode=mode, save=True)
    alone = K.gated_ff(x, wg, wu, wd, act=Activation.SILU, mode=mode)
    return [y, alone, *saved, *K.gated_ff_backward(dy, x, wg, wu, wd, saved, mode=mode)]


def fill_scratch(byte):
    for ws in K._workspaces.values():
        ws.fill_(byte)


KINDS = [("bf16", GemmMode.TF32X3), ("f16", GemmMode.TF32X3)] + [("f32", m) for m in GemmMode]


# f from 1 to 3 past a multiple of 4; k and d odd, even and whole
@pytest.mark.parametrize("kind,mode", KINDS, ids=lambda v: getattr(v, "name", v))
@pytest.mark.parametrize("m", [1, 3, 8, 17, 32, 48, 70, 300])
def test_what_scratch_held_does_not_matter(m, kind, mode):
    for k, f, d in ((1, 1, 1), (64, 129, 40), (33, 262, 7), (72, 203, 129), (130, 516, 64)):
        args = inputs(m, k, f, d, kind, seed=m)
        all_bits(args, mode)  # the workspace has its size
        fill_scratch(0)
        want = all_bits(args, mode)
        fill_scratch(0xFF)
        got = all_bits(args, mode)
        fill_scratch(0xFF)
        again = K.gated_ff(*args[:4], mode=mode)  # a forward pass right behind
        for i, (a, b) in enumerate(zip(got, want)):
            assert torch.isfinite(b).all() and torch.equal(a, b), (i, k, f, d)
        assert torch.equal(again, want[1]), (k, f, d)
    assert K.kernel_status() == 0


@pytest.mark.parametrize("kind", list(TYPES))
def test_not_finite_h_of_an_earlier_call_stays_there(kind):
    """A call whose h is not finite, then one with fewer hidden units whose padding lies
    over it."""
    x, wg, wu, wd, _ = inputs(4, 64, 136, 64, kind)
    clean = K.gated_ff(x, wg[:, :131].contiguous(), wu[:, :131].contiguous(), wd[:131].contiguous())
    K.gated_ff(torch.full_like(x, math.nan), wg, wu, wd)
    again = K.gated_ff(x, wg[:, :131].contiguous(), wu[:, :131].contiguous(), wd[:131].contiguous())
    assert torch.isfinite(clean).all() and torch.equal(clean, again)
