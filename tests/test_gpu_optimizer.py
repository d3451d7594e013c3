"""AdamW over many tensors and the gradient norm, on the GPU: bit for bit against
the float32 restatement, within derived bounds of float64, and where such kernels
go wrong (short, unaligned and many tensors, 8-bit blocks that end inside a
tensor, values that are not finite, graph replays, other streams)."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import _optimizer_ref as R
from zengpu_b200 import Dispatch, kernels as K

pytestmark = pytest.mark.gpu

HYPER = dict(lr=3e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)
REF = dict(lr=3e-3, b1=0.9, b2=0.95, eps=1e-8, wd=0.1)
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def normal(n, seed, scale=1.0):
    return (np.random.default_rng(seed).standard_normal(n) * scale).astype(np.float32)


def cuda(x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x))
    return (t.to(dtype) if dtype else t).cuda()


def host(t):
    t = t.cpu()
    return t.view(torch.uint8).numpy() if t.dtype == torch.float8_e4m3fn else t.float().numpy()


def check_weight(got, want, p0, steps, kind):
    """With 8-bit moments a step's change of the weight is a quotient of approximate
    instructions: the root within 2^-22 of itself, the reciprocal 2^-23, the product
    2^-24, under 2^-21 of the change; the change is at most what the weight moved plus
    decay (counted once more as slack).  Each step then rounds the weight to `kind`,
    half a step (2^-24 of it for f32), and may round to the other neighbour."""
    moved = np.abs(want - p0) + 1e-3 * np.abs(p0) + 1e-2
    half = max(torch.finfo(kind).eps / 2, 2.0 ** -24)
    bound = steps * (2.0 ** -21 * moved + 2 * half * np.abs(want))
    assert np.all(np.abs(got - want) <= bound), np.max(np.abs(got - want) / bound)


class Case:
    """Tensors of `sizes` with moments as after some steps, on the GPU and as float32 copies."""

    def __init__(self, sizes, kind="f32", grad="f32", bits=32, master=False, offset=0):
        def on_gpu(x, dtype=None):  # `offset` elements past an aligned address
            t = cuda(np.concatenate([np.zeros(offset, x.dtype), x]), dtype)
            return t[offset:]
        self.bits, self.kind, self.steps = bits, TYPES[kind], 0
        self.p0 = [normal(n, 10 + i, 0.05) for i, n in enumerate(sizes)]
        self.params = [on_gpu(p, TYPES[kind]) for p in self.p0]
        self.master = [on_gpu(p) for p in self.p0] if master else None
        if not master:
            self.p0 = [host(p) for p in self.params]
        self.grads = [on_gpu(normal(n, 200 + i, 2e-2), TYPES[grad]) for i, n in enumerate(sizes)]
        self.g0 = [host(g) for g in self.grads]
        m = [normal(n, 400 + i, 1e-2) for i, n in enumerate(sizes)]
        r = [np.abs(normal(n, 600 + i, 2e-2)) for i, n in enumerate(sizes)]
        for x in m + r:
            x[::7] = 0
        if bits == 32:
            v = [x * x for x in r]
            self.ref = list(zip(self.p0, m, v, [None] * len(m), [None] * len(m)))
            self.state = {"exp_avg": [on_gpu(x) for x in m], "exp_avg_sq": [on_gpu(x) for x in v]}
        else:
            mq, vq = [R.to_8bit(x) for x in m], [R.to_8bit(x, True) for x in r]
            self.ref = [(p, a[0], b[0], a[1], b[1]) for p, a, b in zip(self.p0, mq, vq)]
            code = lambda x: on_gpu(x).view(torch.float8_e4m3fn)  # noqa: E731
            self.state = {"exp_avg": [code(a[0]) for a in mq], "exp_avg_sq": [code(a[0]) for a in vq],
                          "exp_avg_scale": [cuda(a[1]) for a in mq],
                          "exp_avg_sq_scale": [cuda(a[1]) for a in vq]}
        self.opt = K.AdamW(self.params, self.grads, state_bits=bits, master=self.master,
                           state=self.state)

    def follow(self, step, s=None):
        """One step of the restatement; 16-bit weights without a master are rounded."""
        new = []
        self.steps += 1
        for (p, m, v, ms, vs), g in zip(self.ref, self.g0):
            p, m, v, ms, vs = R.step_f32(p, m, v, g, step, s=s, bits=self.bits, ms=ms, vs=vs, **REF)
            if self.master is None:
                p = host(torch.from_numpy(p).to(self.kind))
            new.append((p, m, v, ms, vs))
        self.ref = new

    def check(self):
        for i, (p, m, v, ms, vs) in enumerate(self.ref):
            w = self.master if self.master is not None else self.params
            if self.bits == 8:
                check_weight(host(w[i]), p, self.p0[i], self.steps,
                             torch.float32 if self.master else self.kind)
                # 16-bit weights beside a master are its rounding
                if self.master is not None:
                    np.testing.assert_array_equal(host(self.params[i]),
                                                  host(self.master[i].to(self.kind)))
            else:
                if self.master is not None:
                    np.testing.assert_array_equal(host(self.master[i]), p)
                np.testing.assert_array_equal(host(self.params[i]),
                                              host(torch.from_numpy(p).to(self.kind)))
            np.testing.assert_array_equal(host(self.state["exp_avg"][i]), m)
            np.testing.assert_array_equal(host(self.state["exp_avg_sq"][i]), v)
            if self.bits == 8:
                np.testing.assert_array_equal(host(self.state["exp_avg_scale"][i]), ms)
                np.testing.assert_array_equal(host(self.state["exp_avg_sq_scale"][i]), vs)


SIZES = [1, 3, 255, 256, 257, 2048, 4096 + 5, 70001]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kind,grad,master", [
    ("f32", "f32", False), ("f32", "bf16", False), ("bf16", "bf16", True), ("bf16", "f32", False),
    ("f16", "f16", True), ("f16", "f16", False), ("bf16", "f16", True)])
def test_adamw_bit_exact(kind, grad, master, bits):
    c = Case(SIZES, kind, grad, bits, master)
    for step in (1, 2, 1000):
        c.opt.step(step, **HYPER)
        c.follow(step)
        c.check()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [1, 2, 4, 7])
def test_adamw_unaligned(offset, bits):
    c = Case([513, 70001], "bf16", "bf16", bits, True, offset)
    c.opt.step(5, **HYPER)
    c.follow(5)
    c.check()


@pytest.mark.parametrize("step", [1, 17, 100000])
def test_adamw_against_float64(step):
    n = 5003
    c = Case([n])
    p, m, v, _, _ = c.ref[0]
    want, off = R.step_f64(p, m, v, c.g0[0], step, **REF)
    c.opt.step(step, **HYPER)
    got = [host(c.params[0]), host(c.state["exp_avg"][0]), host(c.state["exp_avg_sq"][0])]
    for x, y, tol in zip(got, want, off):
        assert np.all(np.abs(x - y) <= tol + 1e-45)


def test_adamw_8bit_against_float64():
    """Codes are within half a step of m and sqrt(v): 2^-4 relative, or half of
    2^-9 of the scale among the subnormal codes (a whole one where the smallest
    code holds a root above zero); 1e-5 covers the float32 roundings before."""
    c = Case([256 * 9 + 17], bits=8)
    p, mq, vq, ms, vs = c.ref[0]
    m, r = R.from_8bit(mq, ms, np.float64), R.from_8bit(vq, vs, np.float64)
    (p1, m1, v1), (tp, _, _) = R.step_f64(p, m, r * r, c.g0[0], 3, **REF)
    c.opt.step(3, **HYPER)
    assert np.all(np.abs(host(c.params[0]) - p1) <= 1.5 * tp)  # v comes through r * r: 2 u more
    for name, x, floor in (("exp_avg", m1, 0.5), ("exp_avg_sq", np.sqrt(v1), 1.0)):
        scale = host(c.state[name + "_scale"][0]).astype(np.float64)
        top = np.abs(R.blocks(x)).max(1)
        np.testing.assert_allclose(scale, top / 448, rtol=1e-6)
        got = R.from_8bit(host(c.state[name][0]), scale, np.float64)
        step = np.repeat(scale, R.BLOCK)[: x.size] * 2.0 ** -9
        assert np.all(np.abs(got - x) <= np.maximum(np.abs(x) / 16, floor * step) + 1e-5 * np.abs(x))
        if name == "exp_avg_sq":
            assert np.all((got > 0) == (x > 0))


def test_adamw_many_tensors_and_empty_ones():
    c = Case([(37 * i) % 700 for i in range(1000)])
    c.opt.step(4, **HYPER)
    c.follow(4)
    c.check()


def test_adamw_leaves_what_lies_around():
    flat = {n: torch.full((1000,), 7.0, device="cuda") for n in ("p", "m", "v")}
    g = torch.ones(333, device="cuda")
    K.AdamW([flat["p"][100:433]], [g], state={"exp_avg": [flat["m"][100:433]],
                                              "exp_avg_sq": [flat["v"][100:433]]}).step(1)
    for t in flat.values():
        assert torch.all(t[:100] == 7) and torch.all(t[433:] == 7) and torch.all(t[100:433] != 7)


def test_adamw_moments_start_at_zero():
    """Step 1 from zero moves each weight by lr against its gradient's sign (eps aside)."""
    for bits in (32, 8):
        p = torch.zeros(1000, device="cuda")
        g = cuda(normal(1000, 1))
        K.AdamW([p], [g], state_bits=bits).step(1, lr=0.5, eps=0.0, weight_decay=0.0)
        np.testing.assert_allclose(host(p), -0.5 * np.sign(host(g)), rtol=1e-6)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_grad_scale(bits):
    c = Case(SIZES, bits=bits)
    c.opt.step(3, grad_scale=torch.tensor([0.37], device="cuda"), **HYPER)
    c.follow(3, s=0.37)
    c.check()
    for bad in (math.nan, math.inf):
        c.opt.step(4, grad_scale=torch.tensor(bad, device="cuda"), **HYPER)
    c.check()


def test_adamw_not_finite():
    """f32 moments: the element alone; 8 bits: its block reads back as NaN, no other."""
    for bits in (32, 8):
        c = Case([1024], bits=bits)
        c.grads[0][300] = math.inf
        c.opt.step(2, **HYPER)
        p = host(c.params[0])
        assert not np.isfinite(p[300]) and np.isfinite(np.delete(p, 300)).all()
        if bits == 8:
            for n in ("exp_avg_scale", "exp_avg_sq_scale"):
                assert np.isnan(host(c.state[n][0])).tolist() == [False, True, False, False]
        else:
            assert np.isfinite(np.delete(host(c.state["exp_avg"][0]), 300)).all()


def test_adamw_tiny_and_large_values():
    """Blocks whose scale would be subnormal, and one near the largest f32."""
    for scale in (1e-42, 1e-30, 1e18):
        c = Case([512], bits=8)
        c.g0[0] = normal(512, 9, scale)
        c.grads[0].copy_(cuda(c.g0[0]))
        for t in c.state.values():
            t[0].view(torch.uint8).zero_()
        c.ref = [(c.ref[0][0], *(np.zeros_like(x) for x in c.ref[0][1:]))]
        c.opt.step(1, **HYPER)
        c.follow(1)
        c.check()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_captured(bits):
    """A captured step reads step, lr and grad_scale from the device at each replay."""
    c = Case(SIZES, "bf16", "bf16", bits, True)
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    lr = torch.zeros(1, device="cuda")
    scale = torch.full((1,), math.nan, device="cuda")
    hyper = {k: v for k, v in HYPER.items() if k != "lr"}
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        c.opt.step(step, lr=lr, grad_scale=scale, **hyper)  # skipped: nothing changes
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step += 1
        c.opt.step(step, lr=lr, grad_scale=scale, **hyper)
    lr.fill_(HYPER["lr"])
    scale.fill_(0.5)
    lr64 = float(lr)  # the f32 the kernel reads
    for t in (1, 2, 3):
        graph.replay()
        new = []
        for (p, m, v, ms, vs), g in zip(c.ref, c.g0):
            new.append(R.step_f32(p, m, v, g, t, s=0.5, bits=bits, ms=ms, vs=vs, **{**REF, "lr": lr64}))
        c.ref, c.steps = new, t
    torch.cuda.synchronize()
    c.check()


def test_adamw_device_step_below_one_changes_nothing():
    c = Case([300])
    for step in (0, -3):
        c.opt.step(torch.full((1,), step, dtype=torch.int64, device="cuda"), **HYPER)
    c.check()


def test_adamw_refusals():
    p, g = torch.zeros(8, device="cuda"), torch.zeros(8, device="cuda")
    opt = K.AdamW([p], [g])
    for bad in (dict(step=0), dict(step=1, beta1=1.0), dict(step=1, beta2=-0.1),
                dict(step=1, eps=-1.0), dict(step=1, lr=math.nan)):
        with pytest.raises(Dispatch):
            opt.step(**bad)
    for bad in (dict(step=torch.ones(1, device="cuda")), dict(step=1, lr=torch.ones(2, device="cuda")),
                dict(step=1, grad_scale=torch.ones(1))):
        with pytest.raises(ValueError):
            opt.step(**bad)
    with pytest.raises(ValueError, match="overlap"):
        K.AdamW([p, p], [g, g])
    with pytest.raises(ValueError, match="overlap"):
        K.AdamW([p], [p])
    with pytest.raises(ValueError, match="overlap"):
        K.AdamW([p[:6], p[4:]], [g[:6], g[:4]])
    K.AdamW([p[:4], p[4:]], [g[:4], g[:4]])  # one gradient for two weights
    with pytest.raises(ValueError, match="master"):
        K.AdamW([p], [g], master=[torch.zeros(8, device="cuda")])
    with pytest.raises(ValueError):
        K.AdamW([p], [g[:4]])
    with pytest.raises(ValueError):
        K.AdamW([torch.zeros(4, 4, device="cuda").t()], [torch.zeros(16, device="cuda")])
    with pytest.raises(ValueError):
        K.AdamW([p], [g], state_bits=16)


# ---- gradient norm -----------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("sizes", [[1], [0, 3, 256], SIZES, [(37 * i) % 700 for i in range(1000)],
                                   [5_000_011, 17]])
def test_grad_norm(sizes, kind):
    grads = [cuda(normal(n, 40 + i, 0.1), TYPES[kind]) for i, n in enumerate(sizes)]
    want = math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))
    norm, scale = K.GradNorm(grads).clip_scale(0.5).tolist()
    # 64-bit sums of n terms: n 2^-53 at most; then one rounding to f32
    assert abs(norm - want) <= 2 ** -24 * want * 1.001
    assert abs(scale - min(1.0, 0.5 / want)) <= 2 ** -24 * 1.001 * min(1.0, 0.5 / want)


def test_grad_norm_edges():
    z = torch.zeros(1000, device="cuda")
    plan = K.GradNorm([z])
    assert plan.clip_scale(1.0).tolist() == [0.0, 1.0]
    z[999] = 3e38  # the square passes f32
    norm, scale = plan.clip_scale(1.0).tolist()
    assert norm == pytest.approx(3e38, rel=1e-6) and scale == pytest.approx(1 / 3e38, rel=1e-6)
    for bad in (math.inf, math.nan):
        z[5] = bad
        norm, scale = plan.clip_scale(1.0).tolist()
        assert not math.isfinite(norm) and math.isnan(scale)
    with pytest.raises(Dispatch):
        plan.clip_scale(0.0)


def test_grad_norm_same_bits_every_time_and_on_two_streams():
    grads = [cuda(normal(3_000_017, i)) for i in range(3)]
    plan = K.GradNorm(grads)
    first = plan.clip_scale(1.0)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    out = []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                out.append(plan.clip_scale(1.0))
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in out)


def test_clipped_step():
    """Norm, factor and step together, with nothing read on the host between."""
    c = Case(SIZES, "bf16", "bf16", 32, True)
    factor = K.GradNorm(c.grads).clip_scale(0.01)
    c.opt.step(1, grad_scale=factor[1:], **HYPER)
    c.follow(1, s=float(factor[1]))
    c.check()
