"""AdamW where eps is tiny: weights without a gradient keep their value, and moments
whose squares are subnormal still count against eps."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import _optimizer_ref as R
from test_gpu_optimizer import host, normal
from zengpu_b200 import kernels as K

pytestmark = pytest.mark.gpu


def plan(p, g, bits, offset=0):
    on = [torch.cat([torch.zeros(offset), torch.from_numpy(t)]).cuda()[offset:] for t in (p, g)]
    return K.AdamW(on[:1], on[1:], state_bits=bits), on[0]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("eps", [1e-300, 1e-50, 1e-45, 1e-40, 1.1e-38, 1.3e-38, 1e-30, 1e-13])
def test_weights_without_a_gradient_only_decay(eps, offset, bits):
    n = 3000
    p, g = normal(n, 1, 0.05), normal(n, 2, 1e-2)
    g[::3] = 0
    opt, got = plan(p, g, bits, offset)
    lr, wd = 3e-3, 0.1
    opt.step(1, lr=lr, beta1=0.9, beta2=0.95, eps=eps, weight_decay=wd)
    got = host(got)
    still = p * np.float32(1 - lr * wd)
    np.testing.assert_array_equal(got[::3], still[::3])
    # the others move by lr against their sign: four roundings of the step and one of the sum
    want = still.astype(np.float64) - lr * np.sign(g)
    u = 2.0 ** -24
    bound = 16 * u * lr + 2 * u * (np.abs(want) + np.abs(still))
    assert np.all((np.abs(got - want) <= bound)[g != 0])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [5e-13, 2e-12, 1e-11, 1e-9])
@pytest.mark.parametrize("beta2", [0.95, 0.9999, 0.9999999])
def test_roots_of_subnormal_moments_count(beta2, eps, bits):
    """v = (1 - beta2) g^2 below f32's smallest normal number, with the root scaled up by
    1 / sqrt(1 - beta2): r root = |g|, next to eps.  From zero the change of the weight is
    all of it.  v has bits down to 2^-149: g is chosen so that a root is within 2^-12 of
    itself, and it counts |g| / (|g| + eps) against the whole."""
    n = 512
    c2 = 1 - beta2
    size = math.sqrt(2.0 ** -127 / c2)
    g = (np.linspace(0.2, 1.0, n) * size).astype(np.float32)
    opt, got = plan(np.zeros(n, np.float32), g, bits)
    opt.step(1, lr=1.0, beta1=0.9, beta2=beta2, eps=eps, weight_decay=0.0)
    g64 = g.astype(np.float64)
    want = -g64 / (g64 + eps)
    share = g64 / (g64 + eps)
    step = 2.0 ** -149 / (c2 * g64 * g64)  # of v, relative: two roundings
    bound = np.abs(want) * (2.0 ** -20 + share * step)
    assert np.all(np.abs(host(got) - want) <= bound), np.max(np.abs(host(got) - want) / bound)


def test_8_bit_steps_with_tiny_eps_follow_the_restatement():
    n = 256 * 5 + 9
    hyper, ref = dict(lr=3e-3, beta1=0.9, beta2=0.95, weight_decay=0.1), dict(lr=3e-3, b1=0.9, b2=0.95, wd=0.1)
    p, g = normal(n, 3, 0.05), normal(n, 4, 2e-2)
    g[::5] = 0
    opt, got = plan(p, g, 8)
    state = (np.zeros(n, np.uint8), np.zeros(n, np.uint8), np.zeros(6, np.float32), np.zeros(6, np.float32))
    for t in (1, 2, 3):
        opt.step(t, eps=1e-40, **hyper)
        p, m, v, ms, vs = R.step_f32(p, state[0], state[1], g, t, bits=8, ms=state[2], vs=state[3],
                                     eps=1e-40, **ref)
        state = (m, v, ms, vs)
        # roots and quotients are exact at such an eps: every bit is the restatement's
        np.testing.assert_array_equal(host(got), p)
        for name, want in zip(("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"), state):
            np.testing.assert_array_equal(host(opt.state[name][0]), want)
