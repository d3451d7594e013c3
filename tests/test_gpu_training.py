"""The feed-forward operators together, as a training loop calls them: forward with
saved products, gradients, norm, clipped AdamW step; through torch tensors, through
DeviceArrays, eager and as one captured graph."""
from __future__ import annotations

import math
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

import _optimizer_ref as R
import zengpu_b200 as zg
from test_gpu_gated_ff import check, inputs, reference
from test_gpu_optimizer import HYPER, REF, check_weight, host
from zengpu_b200 import Activation, kernels as K

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]
NAMES = ("dw_gate", "dw_up", "dw_down")


class Layer:
    """A gated block with its optimiser and gradient buffers, as a program keeps them."""

    def __init__(self, shape, kind, bits):
        self.x, *self.weights, self.dy = inputs(*shape, kind, seed=4)
        self.kind = kind
        self.master = None if kind == "f32" else [w.float() for w in self.weights]
        self.grads = [torch.empty_like(w) for w in self.weights]
        self.opt = K.AdamW(self.weights, self.grads, state_bits=bits, master=self.master)
        self.norm = K.GradNorm(self.grads)

    def step(self, number, act=Activation.SILU, **hyper):
        y, saved = K.gated_ff(self.x, *self.weights, act=act, save=True)
        dx, *_ = K.gated_ff_backward(self.dy, self.x, *self.weights, saved, act=act,
                                     out=(None, *self.grads))
        factor = self.norm.clip_scale(0.5)
        self.opt.step(number, grad_scale=factor[1:], **hyper)
        return y, dx, factor


@pytest.mark.parametrize("kind,bits", [("f32", 32), ("bf16", 8), ("f16", 32)])
@pytest.mark.parametrize("shape", [(192, 128, 264, 128), (33, 65, 101, 47)], ids=str)
def test_training_steps(shape, kind, bits):
    """Each step's parts against their references, from the state the step found."""
    layer = Layer(shape, kind, bits)
    for number in (1, 2, 3):
        before = [w.clone() for w in layer.weights]
        p0 = [host(t).reshape(-1) for t in (layer.master or layer.weights)]
        state = {n: [host(t).reshape(-1) for t in ts] for n, ts in layer.opt.state.items()}
        y, dx, factor = layer.step(number, **HYPER)
        want = reference(layer.x, *before, layer.dy, Activation.SILU)
        got = {"y": y, "dx": dx} | dict(zip(NAMES, layer.grads))
        check(got, want, kind, min(shape) >= 64)
        norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in layer.grads))
        assert abs(float(factor[0]) - norm) <= 1.001 * 2.0 ** -24 * norm
        for i, g in enumerate(layer.grads):
            ms, vs = (state[n][i] for n in ("exp_avg_scale", "exp_avg_sq_scale")) if bits == 8 \
                else (None, None)
            p, m, v, ms, vs = R.step_f32(p0[i], state["exp_avg"][i], state["exp_avg_sq"][i],
                                         host(g).reshape(-1), number, s=float(factor[1]),
                                         bits=bits, ms=ms, vs=vs, **REF)
            new = host((layer.master or layer.weights)[i]).reshape(-1)
            if bits == 8:
                check_weight(new, p, p0[i], 1, torch.float32)
            else:
                np.testing.assert_array_equal(new, p)
            np.testing.assert_array_equal(host(layer.opt.state["exp_avg"][i]).reshape(-1), m)
            np.testing.assert_array_equal(host(layer.opt.state["exp_avg_sq"][i]).reshape(-1), v)
            if layer.master:
                assert torch.equal(layer.weights[i], layer.master[i].to(layer.weights[i].dtype))


@pytest.mark.parametrize("kind,bits", [("f32", 32), ("bf16", 8)])
def test_captured_training_step(kind, bits):
    """A whole step captured once and replayed gives the bits of eager steps, with
    another layer trained eagerly in between on a stream of its own."""
    shape = (160, 128, 520, 128)
    eager, captured, other = (Layer(shape, kind, bits) for _ in range(3))
    for number in (1, 2, 3, 4):
        eager.step(number, **HYPER)
    count = torch.zeros(1, dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        count += 1
        captured.step(count, **HYPER)  # the first step, before the capture
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        count += 1
        captured.step(count, **HYPER)
    torch.cuda.synchronize()
    for number in (1, 2, 3):
        graph.replay()
        with torch.cuda.stream(side):
            other.step(number, **HYPER)
    torch.cuda.synchronize()
    for a, b in zip(eager.weights + (eager.master or []), captured.weights + (captured.master or [])):
        assert torch.equal(a, b)


# ---- DeviceArrays ------------------------------------------------------------------------
DTYPES = {"f32": zg.DType.F32, "f16": zg.DType.F16, "bf16": zg.DType.Bf16}


def put(device, pool, t, dtype):
    raw = t.contiguous().cpu().view(torch.uint8).numpy() if t.dtype != torch.uint8 else t.cpu().numpy()
    a = pool.alloc(list(t.shape), dtype)
    device.write_buffer(a.buffer, 0, raw)
    return a


def get(device, a, like):
    n = a.size_bytes()
    raw = np.empty(n, np.uint8)
    device.read_buffer_async(a.buffer, 0, raw, n).wait(10.0)
    return torch.from_numpy(raw.copy()).view(like.dtype).view(like.shape)


@pytest.mark.parametrize("memory", [zg.MemoryUsage.Upload, zg.MemoryUsage.GpuOnly])
@pytest.mark.parametrize("kind", list(DTYPES))
def test_device_arrays(device, kind, memory):
    """The array calls give the bits of the tensor calls."""
    pool = zg.BufferPool(device, memory)
    host_pool = zg.BufferPool(device)
    gemm, level1 = zg.GemmKernel(device), zg.Level1Kernels(device)
    gemm.mode = zg.GemmMode.TF32X3
    layer = Layer((70, 136, 200, 72), kind, 32)
    master0 = [m.clone() for m in layer.master] if layer.master else None
    dt = DTYPES[kind]
    x, dy = put(device, host_pool, layer.x, dt), put(device, host_pool, layer.dy, dt)
    # weights live where the results do: in-place steps follow their residency
    w = []
    for t in layer.weights:
        a = pool.alloc(list(t.shape), dt)
        device.write_buffer(a.buffer, 0, t.cpu().view(torch.uint8).numpy())
        w.append(a)
    zeros = lambda t: put(device, host_pool, torch.zeros(t.shape), zg.DType.F32)  # noqa: E731
    m, v = [zeros(t) for t in layer.weights], [zeros(t) for t in layer.weights]
    master = [put(device, host_pool, t, zg.DType.F32) for t in master0] if master0 else None
    y, saved = gemm.gated_ff(device, pool, x, *w, act=Activation.GELU, save=True)
    dx, *dw = gemm.gated_ff_backward(device, pool, dy, x, *w, saved, act=Activation.GELU)
    factor = level1.grad_norm(device, pool, dw, 0.5)
    level1.adamw(device, w, dw, m, v, 1, master=master, norm_scale=factor, **HYPER)
    want_y, want_dx, want_factor = layer.step(1, act=Activation.GELU, **HYPER)
    torch.cuda.synchronize()
    assert torch.equal(get(device, y, want_y), want_y.cpu())
    assert torch.equal(get(device, dx, want_dx), want_dx.cpu())
    assert torch.equal(get(device, factor, want_factor), want_factor.cpu())
    for a, t in zip(dw + w, layer.grads + layer.weights):
        assert torch.equal(get(device, a, t), t.cpu())
    for a, t in zip(m + v, layer.opt.state["exp_avg"] + layer.opt.state["exp_avg_sq"]):
        assert torch.equal(get(device, a, t), t.cpu())
    assert gemm.gated_ff(device, pool, x, *w).shape == [70, 72]
    for p in (pool, host_pool):
        p.close()


def test_device_array_8bit_moments(device, pool):
    n = 1000
    p, g = torch.randn(n), torch.randn(n) * 1e-2
    t = [p.cuda()]
    opt = K.AdamW(t, [g.cuda()], state_bits=8)
    opt.step(1, **HYPER)
    opt.step(2, **HYPER)
    arrays = [put(device, pool, x, d) for x, d in (
        (p, zg.DType.F32), (g, zg.DType.F32), (torch.zeros(n, dtype=torch.uint8), zg.DType.U8),
        (torch.zeros(n, dtype=torch.uint8), zg.DType.U8), (torch.zeros(4), zg.DType.F32),
        (torch.zeros(4), zg.DType.F32))]
    pa, ga, ma, va, ms, vs = ([a] for a in arrays)
    level1 = zg.Level1Kernels(device)
    for step in (1, 2):
        level1.adamw(device, pa, ga, ma, va, step, scales=(ms, vs), **HYPER)
    torch.cuda.synchronize()
    assert torch.equal(get(device, pa[0], p), t[0].cpu())
    for a, name in ((ma, "exp_avg"), (va, "exp_avg_sq"), (ms, "exp_avg_scale"),
                    (vs, "exp_avg_sq_scale")):
        like = opt.state[name][0].cpu().view(torch.uint8)
        assert torch.equal(get(device, a[0], like), like)


def test_device_array_refusals(device, pool):
    gemm, level1 = zg.GemmKernel(device), zg.Level1Kernels(device)
    alloc = lambda *shape, dtype=zg.DType.F32: pool.alloc(list(shape), dtype)  # noqa: E731
    x, wg, wu, wd = alloc(4, 8), alloc(8, 16), alloc(8, 16), alloc(16, 8)
    for bad in ((alloc(4, 9), wg, wu, wd), (x, wg, alloc(8, 15), wd), (x, wg, wu, alloc(8, 8)),
                (alloc(4, 8, dtype=zg.DType.F16), wg, wu, wd), (alloc(32), wg, wu, wd),
                (alloc(4, 8, dtype=zg.DType.I32), wg, wu, wd)):
        with pytest.raises(zg.Dispatch):
            gemm.gated_ff(device, pool, *bad)
    free = [pool.free_count(1 << b) for b in range(8, 20)]
    with pytest.raises(zg.Dispatch, match="activation"):
        gemm.gated_ff(device, pool, x, wg, wu, wd, act=9)
    # the outputs of a refused call went back to the pool
    assert sum(pool.free_count(1 << b) for b in range(8, 20)) >= sum(free)
    gone = alloc(8, 16)
    device.destroy_buffer(gone.buffer)
    with pytest.raises(zg.StaleHandle):
        gemm.gated_ff(device, pool, x, gone, wu, wd)
    p, g, m, v = (alloc(64) for _ in range(4))
    with pytest.raises(zg.Dispatch, match="twice"):
        level1.adamw(device, [p], [g], [m], [m], 1)
    with pytest.raises(zg.Dispatch, match="twice"):
        level1.adamw(device, [p], [p], [m], [v], 1)
    with pytest.raises(zg.Dispatch, match="scales"):
        level1.adamw(device, [p], [g], [alloc(64, dtype=zg.DType.U8)],
                     [alloc(64, dtype=zg.DType.U8)], 1)
    with pytest.raises(zg.Dispatch, match="shape"):
        level1.adamw(device, [p], [alloc(63)], [m], [v], 1)
    with pytest.raises(zg.Dispatch):
        level1.adamw(device, [p], [g], [m], [v], 0)
    with pytest.raises(zg.Dispatch):
        level1.grad_norm(device, pool, [alloc(4, dtype=zg.DType.I32)], 1.0)
    with pytest.raises(ValueError):
        level1.adamw(device, [p], [g, g], [m], [v], 1)


FIRST = """
import torch
from zengpu_b200 import kernels as K
x, wg, wu, wd, dy = (torch.randn(s, device="cuda").to({kind}) * 0.1
                     for s in ((m, 64), (64, 136), (64, 136), (136, 64), (m, 64)))
grads = [torch.empty_like(w) for w in (wg, wu, wd)]
opt, norm = K.AdamW([w.clone() for w in (wg, wu, wd)], grads, state_bits=8), K.GradNorm(grads)
torch.cuda.synchronize()
def run():
    y, saved = K.gated_ff(x, wg, wu, wd, save=True)
    K.gated_ff_backward(dy, x, wg, wu, wd, saved, out=(None, *grads))
    opt.step(1, grad_scale=norm.clip_scale(1.0)[1:])
    return y
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = run()
y.zero_()
graph.replay()
torch.cuda.synchronize()
assert torch.equal(y, K.gated_ff(x, wg, wu, wd)) and K.kernel_status() == 0
"""


@pytest.mark.parametrize("kind,m", [("torch.bfloat16", 5), ("torch.float16", 300),
                                    ("torch.float32", 5), ("torch.float32", 300)])
def test_first_call_of_a_process_may_be_captured(kind, m):
    """Kernels load and attributes are set at the first call; a capture takes that too."""
    code = FIRST.replace("{kind}", kind).replace("(m, 64)", f"({m}, 64)")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
