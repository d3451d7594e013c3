"""The gated feed-forward block and its gradients on the GPU, against float64.

Bounds.  u = eps / 2 of the tensors' type is the most one rounding is off,
relative to the value.  With 16-bit tensors y and every gradient see two: one of
an operand (h, dg, du), one of the result; spread evenly within a half step each
has an rms of at most u / sqrt(3), so the relative Frobenius error is at most
sqrt(2 / 3) u for long sums of independent terms: u is the bar.  Element by
element nothing averages: |error| <= u |result| + the sum of u |operand| |factor|,
plus what the f32 sums lose, (n + 8) 2^-23 of the sum of magnitudes over n terms
(the tensor core's additions truncate; 8 covers the activation's few ulps)."""
from __future__ import annotations

import math

import pytest
import torch

from zengpu_b200 import Activation, Dispatch, GemmMode, kernels as K

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ACTS = list(Activation)


def inputs(m, k, f, d, kind, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(TYPES[kind])
    return (normal(m, k), normal(k, f, scale=1.3 / math.sqrt(k)), normal(k, f, scale=k ** -0.5),
            normal(f, d, scale=f ** -0.5), normal(m, d))


def act64(g, act):
    """The activation and its slope from their definitions, in float64."""
    if act == Activation.RELU:
        return torch.where(g > 0, g, 0.0), (g > 0).double()
    if act == Activation.SILU:
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    if act == Activation.GELU:
        c = torch.special.erfc(-g / math.sqrt(2)) / 2  # 1 + erf would cancel in the left tail
        return g * c, c + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    q = math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
    c = torch.sigmoid(2 * q)  # (1 + tanh q) / 2, which would cancel
    slope = 2 * c * torch.sigmoid(-2 * q) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * g * g)
    return g * c, c + g * slope


def reference(x, wg, wu, wd, dy, act):
    """{name: (value, magnitude of what enters its last product, sum of rounded operands)}."""
    x, wg, wu, wd, dy = (t.double() for t in (x, wg, wu, wd, dy))
    g, u = x @ wg, x @ wu
    a, slope = act64(g, act)
    h, dh = a * u, dy @ wd.t()
    dg, du = dh * u * slope, dh * a
    # f32 sums that enter h, dg, du: errors of g, u, dh in units of 2^-23, by magnitudes
    eg, eu = x.abs() @ wg.abs(), x.abs() @ wu.abs()
    ed = dy.abs() @ wd.abs().t()
    n, nd = x.shape[1] + 8, wd.shape[1] + 8
    # 1.13 bounds the slopes, 0.8 their change per unit (relu's step aside, see the callers)
    oh = n * (1.13 * eg * u.abs() + a.abs() * eu) + 8 * h.abs()
    odu = nd * ed * a.abs() + n * 1.13 * eg * dh.abs() + 8 * du.abs()
    odg = nd * ed * (u * slope).abs() + n * dh.abs() * (eu * slope.abs() + 0.8 * eg * u.abs()) \
        + 8 * dg.abs()
    t = lambda z: z.t()  # noqa: E731
    out = {"y": (h @ wd, h.abs() @ wd.abs(), oh @ wd.abs(), h.shape[1]),
           "dx": (dg @ wg.t() + du @ wu.t(), dg.abs() @ wg.abs().t() + du.abs() @ wu.abs().t(),
                  odg @ wg.abs().t() + odu @ wu.abs().t(), 2 * h.shape[1]),
           "dw_gate": (t(x) @ dg, t(x).abs() @ dg.abs(), t(x).abs() @ odg, x.shape[0]),
           "dw_up": (t(x) @ du, t(x).abs() @ du.abs(), t(x).abs() @ odu, x.shape[0]),
           "dw_down": (t(h) @ dy, t(h).abs() @ dy.abs(), t(oh) @ dy.abs(), x.shape[0])}
    return out


def rel_fro(x, y):
    return float((x.double() - y).norm() / y.norm().clamp_min(1e-300))


def check(got, want, kind, long_sums):
    u = torch.finfo(TYPES[kind]).eps / 2
    tiny = torch.finfo(TYPES[kind]).smallest_normal * torch.finfo(TYPES[kind]).eps
    for name, t in got.items():
        value, size, inner, n = want[name]
        bound = u * value.abs() + u * size + 2.0 ** -23 * (inner + (n + 8) * size)
        bound += tiny * (1 + n)  # f16 and bf16 below their normal range
        assert torch.isfinite(t).all(), name
        worst = float(((t.double() - value).abs() / bound).max())
        assert worst <= 1.0, (name, worst)
        if long_sums:
            bar = u if kind != "f32" else 2e-6
            assert rel_fro(t, value) <= bar, (name, rel_fro(t, value))


def run_all(args, act, mode=GemmMode.TF32X3):
    x, wg, wu, wd, dy = args
    y, saved = K.gated_ff(x, wg, wu, wd, act=act, mode=mode, save=True)
    dx, dwg, dwu, dwd = K.gated_ff_backward(dy, x, wg, wu, wd, saved, act=act, mode=mode)
    return {"y": y, "dx": dx, "dw_gate": dwg, "dw_up": dwu, "dw_down": dwd}


# m, k, f, d: single elements, odd sizes, either side of the tiles' edges, few rows over
# long sums, many rows over short ones
SHAPES = [(1, 1, 1, 1), (1, 8, 8, 8), (3, 5, 7, 9), (1, 2048, 4096, 1024), (2, 64, 136, 520),
          (8, 1024, 2048, 768), (16, 512, 1000, 512), (17, 64, 64, 64), (48, 1024, 2816, 1024),
          (64, 640, 1280, 640), (65, 72, 200, 40), (100, 256, 256, 256), (128, 512, 1024, 512),
          (130, 1000, 333, 77), (255, 128, 128, 136), (257, 256, 520, 264), (300, 2048, 640, 1024),
          (513, 96, 256, 2056), (1025, 264, 1288, 256), (2500, 16, 24, 8)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_float64(shape, kind):
    args = inputs(*shape, kind)
    act = Activation.SILU
    got = run_all(args, act)
    x, wg, wu, wd, _ = args
    assert torch.equal(K.gated_ff(x, wg, wu, wd, act=act), got["y"])  # saving changes nothing
    check(got, reference(*args, act), kind, min(shape) >= 64)
    assert K.kernel_status() == 0


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("act", ACTS, ids=lambda a: a.name)
@pytest.mark.parametrize("shape", [(5, 128, 264, 136), (200, 192, 456, 320)], ids=str)
def test_activations(shape, act, kind):
    args = inputs(*shape, kind, seed=3)
    if act == Activation.RELU:  # keep g away from the step, where its sign is the sums' last bit
        x, wg = args[0].float(), args[1].float()
        assert float((x.double() @ wg.double()).abs().min()) > 0
    check(run_all(args, act), reference(*args, act), kind, min(shape) >= 64)


@pytest.mark.parametrize("act", ACTS, ids=lambda a: a.name)
def test_saved_and_activation_tails(act):
    """g from -30 to 30 through identity weights: `saved` is exact there, and each
    activation holds its relative accuracy in the tails (2^-20: some ulps of e^-g)."""
    n = 512
    eye = torch.eye(n, device="cuda")
    g = torch.linspace(-30, 30, n, device="cuda").repeat(4, 1).contiguous()
    y, (pre_g, pre_u) = K.gated_ff(g, eye, eye, eye, act=act, save=True)
    tol = 2.0 ** -20
    assert rel_fro(pre_g, g.double()) <= tol and torch.equal(pre_g, pre_u)
    want = act64(pre_g.double(), act)[0] * pre_u.double()
    # GELU's e^(-g^2/2) turns 2^-24 of g^2 / 2 = 450 into 2^-15; results under 1e-30 aside
    far = want.abs() > 1e-30
    loose = 2.0 ** -13 if act in (Activation.GELU, Activation.GELU_TANH) else 2.0 ** -18
    assert torch.all((y.double() - want).abs()[far] <= loose * want.abs()[far])


@pytest.mark.parametrize("mode,bar", [(GemmMode.SIMT_FP32, 2e-6), (GemmMode.TF32X3, 2e-6),
                                      (GemmMode.TF32_BF16X2, 3e-5), (GemmMode.BF16X3, 3e-5),
                                      (GemmMode.TF32, 1.5e-2)], ids=lambda v: getattr(v, "name", ""))
@pytest.mark.parametrize("shape", [(300, 520, 1000, 264), (130, 77, 201, 55)], ids=str)
def test_f32_modes(shape, mode, bar):
    """Three products follow one another at most: three times sgemm's bar for a mode
    (TF32X3 sums shorter runs here and stays within a few ulps)."""
    args = inputs(*shape, "f32", seed=5)
    got = run_all(args, Activation.SILU, mode)
    want = reference(*args, Activation.SILU)
    for name, t in got.items():
        assert rel_fro(t, want[name][0]) <= bar, (name, rel_fro(t, want[name][0]))


@pytest.mark.parametrize("act", [Activation.SILU, Activation.GELU, Activation.GELU_TANH],
                         ids=lambda a: a.name)
def test_gradients_against_differences(act):
    """(L(w + e v) - L(w - e v)) / 2e along random directions, L = sum(y dy): the f32
    noise of L (2^-22 of its terms' size) over 2e, and e^2 / 6 of a third derivative."""
    args = list(inputs(40, 64, 96, 72, "f32", seed=9))
    got = run_all(args, act, GemmMode.SIMT_FP32)
    gen = torch.Generator(device="cuda").manual_seed(1)
    e = 2e-3
    for i, name in ((0, "dx"), (1, "dw_gate"), (2, "dw_up"), (3, "dw_down")):
        v = torch.randn(args[i].shape, generator=gen, device="cuda")
        v = v * (args[i].norm() / v.norm())
        def loss(s):
            moved = list(args)
            moved[i] = args[i] + s * v
            y = K.gated_ff(*moved[:4], act=act, mode=GemmMode.SIMT_FP32)
            return float((y.double() * args[4].double()).sum())
        slope = (loss(e) - loss(-e)) / (2 * e)
        want = float((got[name].double() * v.double()).sum())
        size = float(got[name].double().norm() * v.double().norm())
        assert abs(slope - want) <= 2e-3 * size, (name, slope, want)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("m", [2, 40, 300])
def test_not_finite_rows_stay_in_their_rows(m, kind):
    x, wg, wu, wd, dy = inputs(m, 128, 256, 128, kind)
    x[m // 2, 3] = math.nan
    dy[m - 1, 5] = math.inf
    y, saved = K.gated_ff(x, wg, wu, wd, save=True)
    bad = torch.zeros(m, dtype=torch.bool, device="cuda")
    bad[m // 2] = True
    assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all()
    dx = K.gated_ff_backward(dy, x, wg, wu, wd, saved)[0]
    bad[m - 1] = True
    assert not torch.isfinite(dx[bad]).any() and torch.isfinite(dx[~bad]).all()


@pytest.mark.parametrize("kind", list(TYPES))
def test_given_outputs_and_what_lies_around(kind):
    """Outputs in the middle of larger buffers, 2 or 4 bytes off a 16-byte boundary."""
    m, k, f, d = 70, 136, 264, 72
    args = inputs(m, k, f, d, kind)
    want = run_all(args, Activation.SILU)
    x, wg, wu, wd, dy = args
    def inside(shape):
        n = math.prod(shape)
        flat = torch.full((n + 200,), 7.0, dtype=TYPES[kind], device="cuda")
        return flat, flat[101:101 + n].view(shape)
    flats, outs = zip(*[inside(s) for s in ((m, d), (m, k), (k, f), (k, f), (f, d))])
    y, saved = K.gated_ff(x, wg, wu, wd, save=True, out=outs[0])
    got = K.gated_ff_backward(dy, x, wg, wu, wd, saved, out=outs[1:])
    assert y is outs[0] and all(a is b for a, b in zip(got, outs[1:]))
    for flat, out, name in zip(flats, outs, ("y", "dx", "dw_gate", "dw_up", "dw_down")):
        assert torch.equal(out, want[name]), name
        assert torch.all(flat[:101] == 7) and torch.all(flat[101 + out.numel():] == 7), name


@pytest.mark.parametrize("m", [1, 33, 200])
def test_unaligned_views(m):
    def shifted(t):
        flat = torch.empty(t.numel() + 8, dtype=t.dtype, device="cuda")
        flat[3:3 + t.numel()].copy_(t.reshape(-1))
        return flat[3:3 + t.numel()].view(t.shape)
    args = inputs(m, 128, 256, 64, "bf16")
    want = run_all(args, Activation.GELU)
    got = run_all([shifted(t) for t in args], Activation.GELU)
    assert all(torch.equal(got[n], want[n]) for n in want)


def test_no_rows():
    x, wg, wu, wd, dy = inputs(0, 64, 128, 32, "bf16")
    y, saved = K.gated_ff(x, wg, wu, wd, save=True)
    assert y.shape == (0, 32) and saved[0].shape == (0, 128)
    dx, *dw = K.gated_ff_backward(dy, x, wg, wu, wd, saved)
    assert dx.shape == (0, 64) and all(torch.all(t == 0) for t in dw)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", [(1, 512, 1024, 512), (24, 256, 1032, 264), (400, 512, 776, 256)],
                         ids=str)
def test_same_bits_on_streams_and_in_graphs(shape, kind):
    """Calls on two streams at once, and a captured pass replayed beside eager ones,
    give the bits of a call alone."""
    args = inputs(*shape, kind)
    want = run_all(args, Activation.SILU)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(run_all(args, Activation.SILU))
    torch.cuda.synchronize()
    graphs, held = [], []
    for s in streams:  # two graphs, captured on the same stream, replayed on two
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(run_all(args, Activation.SILU))
        graphs.append(g)
    for o in held:
        for t in o.values():
            t.zero_()
    torch.cuda.synchronize()
    for _ in range(2):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        outs.append(run_all(args, Activation.SILU))
    torch.cuda.synchronize()
    for o in outs + held:
        assert all(torch.equal(o[n], want[n]) for n in want)
    assert K.kernel_status() == 0


def test_offsets_past_32_bits():
    """m f over 2^31: the last rows are computed, and land, where they belong."""
    m, k, f, d = 140_000, 16, 16_384, 16
    x, wg, wu, wd, dy = inputs(m, k, f, d, "bf16")
    y, saved = K.gated_ff(x, wg, wu, wd, save=True)
    dx, *dw = K.gated_ff_backward(dy, x, wg, wu, wd, saved)
    rows = torch.tensor([0, 65535, 131_072, m - 1], device="cuda")
    part = (x[rows], wg, wu, wd, dy[rows])
    want = reference(*part, Activation.SILU)
    check({"y": y[rows], "dx": dx[rows]}, want, "bf16", False)
    half = m // 2  # each weight gradient is the sum of those of two halves of the rows
    parts = [K.gated_ff_backward(dy[a:b], x[a:b], wg, wu, wd, tuple(t[a:b] for t in saved))[1:]
             for a, b in ((0, half), (half, m))]
    for whole, a, b in zip(dw, *parts):
        # three roundings to bf16 of values of these sizes
        size = whole.double().abs() + a.double().abs() + b.double().abs()
        assert torch.all((whole.double() - a.double() - b.double()).abs() <= 2.0 ** -8 * size + 0.5)


def test_refusals():
    x, wg, wu, wd, dy = inputs(4, 16, 32, 8, "bf16")
    for bad in ((x.t().contiguous().t(), wg, wu, wd), (x, wg[:, :24], wu, wd),
                (x, wg, wu, wd.t()), (x.float(), wg, wu, wd), (x[0], wg, wu, wd),
                (x.cpu(), wg, wu, wd), (x.double(), wg, wu, wd), (x, wg, wu.half(), wd)):
        with pytest.raises(ValueError):
            K.gated_ff(*bad)
    with pytest.raises(ValueError):
        K.gated_ff(x, wg, wu, wd, out=torch.empty(4, 9, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(Dispatch, match="activation"):
        K.gated_ff(x, wg, wu, wd, act=7)
    with pytest.raises(Dispatch, match="mode"):
        K.gated_ff(*(t.float() for t in (x, wg, wu, wd)), mode=9)
    with pytest.raises(Dispatch, match="shape"):
        K.gated_ff(x[:, :0].contiguous(), wg[:0], wu[:0], wd)
    y, saved = K.gated_ff(x, wg, wu, wd, save=True)
    for bad in ((saved[0],), (saved[0], None), (saved[0].half(), saved[1])):
        with pytest.raises(ValueError):
            K.gated_ff_backward(dy, x, wg, wu, wd, bad)
    with pytest.raises(ValueError):
        K.gated_ff_backward(dy[:3], x, wg, wu, wd, saved)
