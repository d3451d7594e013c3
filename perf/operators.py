"""Feed-forward layers of a language model: the gated block, its gradients, and the step that trains its weights.

Four operators, each with a plain form in elementary torch operations and, where ``own`` is true, this library's calls:

* ``forward``  y = (act(x w_gate) * (x w_up)) w_down, one token or a batch of them;
* ``train``    the same with the four gradients of y against dy;
* ``adamw``    one AdamW step over all weights of several layers, moments in 32 or in 8 bits;
* ``norm``     the 2-norm over all gradients and the factor that clips them to a largest norm.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LR, BETA1, BETA2, EPS, DECAY = 3e-4, 0.9, 0.95, 1e-8, 0.1
MAX_NORM = 1.0
BLOCK = 256  # elements that share a scale where moments are held in 8 bits
E4M3_MAX, E4M3_MIN = 448.0, 2.0 ** -9
TINY = 2.0 ** -126


# ---- cases -------------------------------------------------------------------------------------
def _ff(name, op, m, k, f, kind, act):
    case = {"op": op, "m": m, "k": k, "f": f, "type": kind, "act": act}
    return dict(case, name=name) if name else case


def _adamw(name, layers, k, f, kind, grad, bits, master):
    case = {"op": "adamw", "layers": layers, "k": k, "f": f, "type": kind, "grad": grad, "bits": bits, "master": master}
    return dict(case, name=name) if name else case


def _norm(name, layers, k, f, grad):
    case = {"op": "norm", "layers": layers, "k": k, "f": f, "grad": grad}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one token through a small layer: a draft model or a test bench, where latency counts
        _ff("forward_token_small", "forward", 1, 1024, 4096, "bf16", "silu"),
        # one token through a wide layer: every weight is read once
        _ff("forward_token", "forward", 1, 4096, 12288, "bf16", "silu"),
        # tokens of many requests decoded together
        _ff("forward_batch", "forward", 48, 4096, 12288, "f16", "silu"),
        # a long prompt, or the evaluation of a 4096-row batch
        _ff("forward_long", "forward", 4096, 4096, 8192, "bf16", "gelu_tanh"),
        # a training step's layer, 16-bit weights
        _ff("train_bf16", "train", 4096, 4096, 8192, "bf16", "silu"),
        # ragged batch through a layer with odd sizes
        _ff("train_odd", "train", 517, 1000, 2605, "f16", "gelu"),
        # the library's own type
        _ff("train_f32", "train", 2048, 1024, 4096, "f32", "silu"),
        # all weights of eight layers in the library's own type
        _adamw("adamw_f32", 8, 2048, 5632, "f32", "f32", 32, False),
        # 16-bit weights with 32-bit masters, moments in 8 bits
        _adamw("adamw_8bit", 8, 2048, 5632, "bf16", "bf16", 8, True),
        # one small layer with odd sizes: the launch counts
        _adamw("adamw_small", 1, 96, 301, "f32", "f32", 32, False),
        # clipping before the step
        _norm("norm_long", 8, 2048, 5632, "bf16"),
        _norm("norm_small", 2, 200, 533, "f32"),
    ]


MOST_FLOPS = {"forward": 6 * 4096 * 4096 * 8192, "train": 18 * 4096 * 4096 * 8192}
MOST_ELEMENTS = 8 * 3 * 2048 * 5632


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["forward", "forward", "train", "train", "adamw", "adamw", "norm"])
    if op in MOST_FLOPS:
        while True:
            m = _log(rng, 1 if op == "forward" else 64, 4096)
            k, f = _log(rng, 256, 4096), _log(rng, 512, 12288)
            if rng.random() < 0.7:  # layers are mostly made of multiples of 64
                k, f = max(64, k // 64 * 64), max(64, f // 64 * 64)
            kind = rng.choice(["bf16", "bf16", "f16", "f32"])
            work = (6 if op == "forward" else 18) * m * k * f
            if work <= MOST_FLOPS[op] // (8 if kind == "f32" else 1):
                return _ff("", op, m, k, f, kind, rng.choice(["silu", "gelu", "gelu_tanh", "relu"]))
    while True:
        layers, k, f = rng.randint(1, 12), _log(rng, 48, 2560), _log(rng, 100, 8192)
        if layers * 3 * k * f <= MOST_ELEMENTS:
            break
    if op == "norm":
        return _norm("", layers, k, f, rng.choice(["f32", "bf16", "f16"]))
    kind, grad = rng.choice([("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16")])
    return _adamw("", layers, k, f, kind, grad, rng.choice([32, 8]), kind != "f32" and rng.random() < 0.7)


def _sizes(case):
    """Elements of each tensor: per layer the gate, up and down weights and a vector of norm weights."""
    k, f = case["k"], case["f"]
    return [k * f, k * f, f * k, k] * case["layers"]


def work(case):
    op = case["op"]
    if op in ("forward", "train"):
        m, k, f = case["m"], case["k"], case["f"]
        size = TYPES[case["type"]].itemsize
        weights, acts = 3 * k * f, 2 * m * k
        if op == "forward":
            return {"bytes": size * (weights + acts), "flops": 6 * m * k * f}
        return {"bytes": size * 2 * (weights + acts), "flops": 18 * m * k * f}
    n = sum(_sizes(case))
    if op == "norm":
        return {"bytes": n * TYPES[case["grad"]].itemsize, "flops": 2 * n}
    moments = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    kind = TYPES[case["type"]].itemsize
    param = kind + 8 if case["master"] else 2 * kind
    return {"bytes": n * (param + TYPES[case["grad"]].itemsize + moments), "flops": 16 * n}


# ---- inputs ------------------------------------------------------------------------------------
def _randn(gen, shape, kind, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(TYPES[kind])


def _flat(case):
    """Where each tensor starts in a flat buffer (a multiple of BLOCK), and the buffer's length."""
    starts, end = [], 0
    for n in _sizes(case):
        starts.append(end)
        end += -(-n // BLOCK) * BLOCK
    return starts, end


def _views(flat, case, per=1):
    """The tensors of a flat buffer that holds one value for `per` elements."""
    return [flat[s // per: s // per + -(-n // per)] for s, n in zip(_flat(case)[0], _sizes(case))]


def _filled(gen, case, scale):
    """A flat f32 buffer of normal values, another spread in each tensor, and zeros between the tensors."""
    flat = torch.zeros(_flat(case)[1], device="cuda")
    for i, t in enumerate(_views(flat, case)):
        t.normal_(0.0, scale * (0.5 + (i * 7 % 5) / 4), generator=gen)
    return flat


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    state = dict(case)
    if op in ("forward", "train"):
        m, k, f, kind = case["m"], case["k"], case["f"], case["type"]
        state["x"] = _randn(gen, (m, k), kind)
        state["w_gate"] = _randn(gen, (k, f), kind, 1.2 / math.sqrt(k))
        state["w_up"] = _randn(gen, (k, f), kind, 1.0 / math.sqrt(k))
        state["w_down"] = _randn(gen, (f, k), kind, 1.0 / math.sqrt(f))
        if op == "train":
            state["dy"] = _randn(gen, (m, k), kind)
        return state
    state["grad_flat"] = _filled(gen, case, 1e-3).to(TYPES[case["grad"]])
    grads = _views(state["grad_flat"], case)
    if op == "norm":
        if own:
            from zengpu_b200 import kernels as K
            state["plan"] = K.GradNorm(grads)
        return state
    weights = _filled(gen, case, 0.02)
    state["param"] = weights.to(TYPES[case["type"]]) if case["type"] != "f32" else weights
    if case["master"]:
        state["master_flat"] = weights
    first, second = _filled(gen, case, 4e-4), _filled(gen, case, 1e-3).square_()
    if case["bits"] == 32:
        state["exp_avg"], state["exp_avg_sq"] = first, second
    else:
        state["exp_avg"], state["exp_avg_scale"] = _to_8bit(first)
        state["exp_avg_sq"], state["exp_avg_sq_scale"] = _to_8bit(second.sqrt_(), positive=True)
    state["step"] = 100
    if own:
        from zengpu_b200 import kernels as K
        moments = {n: _views(state[n], case, BLOCK if n.endswith("scale") else 1)
                   for n in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale") if n in state}
        state["plan"] = K.AdamW(_views(state["param"], case), grads, state_bits=case["bits"],
                                master=_views(weights, case) if case["master"] else None, state=moments)
    return state


# ---- the operators -----------------------------------------------------------------------------
def _act(g, act):
    """The activation and its derivative."""
    if act == "relu":
        on = (g > 0).to(g.dtype)
        return g * on, on
    if act == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


def _plain_forward(s):
    x, wg, wu, wd = (s[n].float() for n in ("x", "w_gate", "w_up", "w_down"))
    y = (_act(x @ wg, s["act"])[0] * (x @ wu)) @ wd
    return {"y": y.to(s["x"].dtype)}


def _plain_train(s):
    x, wg, wu, wd, dy = (s[n].float() for n in ("x", "w_gate", "w_up", "w_down", "dy"))
    g, u = x @ wg, x @ wu
    a, slope = _act(g, s["act"])
    h = a * u
    dh = dy @ wd.t()
    dg, du = dh * u * slope, dh * a
    out = {"y": h @ wd, "dx": dg @ wg.t() + du @ wu.t(), "dw_gate": x.t() @ dg, "dw_up": x.t() @ du, "dw_down": h.t() @ dy}
    return {n: t.to(s["x"].dtype) for n, t in out.items()}


def _to_8bit(x, positive=False):
    """Codes in e4m3 and one f32 scale for each BLOCK; with `positive`, no value over zero becomes zero."""
    x = x.view(-1, BLOCK)
    top = x.abs().amax(1, keepdim=True)
    scale = torch.where(top > 0, (top * (1 / E4M3_MAX)).clamp_min(TINY), top)
    q = x * torch.where(top > 0, 1 / scale, top)
    if positive:
        q = torch.where(x > 0, q.clamp_min(E4M3_MIN), q)
    return q.to(torch.float8_e4m3fn).view(-1), scale.view(-1)


def _from_8bit(q, scale):
    return (q.float().view(-1, BLOCK) * scale.view(-1, 1)).view(-1)


def _plain_adamw(s):
    s["step"] += 1
    step_size = LR / (1 - BETA1 ** s["step"])
    root = 1 / math.sqrt(1 - BETA2 ** s["step"])
    g = s["grad_flat"].float()
    p = s["master_flat"] if s["master"] else s["param"].float()
    if s["bits"] == 32:
        m, v = s["exp_avg"], s["exp_avg_sq"]
    else:
        m = _from_8bit(s["exp_avg"], s["exp_avg_scale"])
        v = _from_8bit(s["exp_avg_sq"], s["exp_avg_sq_scale"]).square_()
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + g * (1 - BETA2) * g
    r = torch.sqrt(v)
    p = p * (1 - LR * DECAY) - m * step_size / (r * root + EPS)
    if s["master"]:
        s["master_flat"].copy_(p)
    s["param"].copy_(p)
    if s["bits"] == 32:
        s["exp_avg"].copy_(m)
        s["exp_avg_sq"].copy_(v)
    else:
        q, scale = _to_8bit(m)
        s["exp_avg"].copy_(q), s["exp_avg_scale"].copy_(scale)
        q, scale = _to_8bit(r, positive=True)
        s["exp_avg_sq"].copy_(q), s["exp_avg_sq_scale"].copy_(scale)
    return _adamw_out(s)


def _adamw_out(s):
    names = ("param", "master_flat", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")
    return {n: s[n] for n in names if n in s}


def _plain_norm(s):
    norm = torch.sqrt(s["grad_flat"].double().square().sum())
    return {"norm": norm.float(), "scale": (MAX_NORM / norm).clamp(max=1.0).float()}


def run(state):
    op = state["op"]
    if not own:
        return {"forward": _plain_forward, "train": _plain_train, "adamw": _plain_adamw, "norm": _plain_norm}[op](state)
    from zengpu_b200 import Activation
    from zengpu_b200 import kernels as K
    if op == "forward":
        return {"y": K.gated_ff(state["x"], state["w_gate"], state["w_up"], state["w_down"], act=Activation[state["act"].upper()])}
    if op == "train":
        act = Activation[state["act"].upper()]
        weights = (state["w_gate"], state["w_up"], state["w_down"])
        y, saved = K.gated_ff(state["x"], *weights, act=act, save=True)
        dx, dw_gate, dw_up, dw_down = K.gated_ff_backward(state["dy"], state["x"], *weights, saved, act=act)
        return {"y": y, "dx": dx, "dw_gate": dw_gate, "dw_up": dw_up, "dw_down": dw_down}
    if op == "adamw":
        state["step"] += 1
        state["plan"].step(state["step"], lr=LR, beta1=BETA1, beta2=BETA2, eps=EPS, weight_decay=DECAY)
        return _adamw_out(state)
    norm_scale = state["plan"].clip_scale(MAX_NORM)
    return {"norm": norm_scale[0], "scale": norm_scale[1]}


# ---- the definition in 64 bits -------------------------------------------------------------------
def _exact_ff(case, seed):
    s = prepare(case, seed)
    names = ("x", "w_gate", "w_up", "w_down")
    x, wg, wu, wd = (s[n].double().requires_grad_(case["op"] == "train") for n in names)
    F = torch.nn.functional
    act = {"silu": F.silu, "relu": F.relu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}[case["act"]]
    y = torch.mm(act(torch.mm(x, wg)).mul(torch.mm(x, wu)), wd)
    if case["op"] == "forward":
        return {"y": y}
    dx, dwg, dwu, dwd = torch.autograd.grad(y, (x, wg, wu, wd), s["dy"].double())
    return {"y": y.detach(), "dx": dx, "dw_gate": dwg, "dw_up": dwu, "dw_down": dwd}


def _exact_codes(x, scale):
    """The e4m3 value nearest to x / scale for each value of blocks x, ties to the even code."""
    codes = [(i & 7) * 2.0 ** -9 if i < 8 else (8 + (i & 7)) * 2.0 ** ((i >> 3) - 10) for i in range(127)]
    table = torch.tensor(codes, dtype=torch.float64, device=x.device)
    between = (table[1:] + table[:-1]) / 2
    q = torch.where(scale > 0, x.abs() / scale, x.abs())
    low, high = torch.bucketize(q, between), torch.bucketize(q, between, right=True)
    pick = torch.where(low % 2 == 0, low, high)  # low < high only at a tie
    return torch.sign(x) * table[pick]


def _exact_adamw(case, seed):
    s = prepare(case, seed)
    t = s["step"] + 1
    out = {n: torch.empty(v.numel(), dtype=torch.float64, device="cuda") for n, v in _adamw_out(s).items()}
    many = 1 << 25
    for a in range(0, s["param"].numel(), many):
        one, few = slice(a, a + many), slice(a // BLOCK, (a + many) // BLOCK)
        g = s["grad_flat"][one].double()
        p = (s["master_flat"] if case["master"] else s["param"])[one].double()
        m, v = s["exp_avg"][one].double(), s["exp_avg_sq"][one].double()
        if case["bits"] == 8:
            m = (m.view(-1, BLOCK) * s["exp_avg_scale"][few].double()[:, None]).view(-1)
            v = (v.view(-1, BLOCK) * s["exp_avg_sq_scale"][few].double()[:, None]).view(-1) ** 2
        m = torch.lerp(g, m, BETA1)
        v = torch.lerp(g * g, v, BETA2)
        p = p - LR * DECAY * p - LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
        out["param"][one] = p
        if case["master"]:
            out["master_flat"][one] = p
        if case["bits"] == 32:
            out["exp_avg"][one], out["exp_avg_sq"][one] = m, v
            continue
        for n, x in (("exp_avg", m.view(-1, BLOCK)), ("exp_avg_sq", v.sqrt().view(-1, BLOCK))):
            scale = x.abs().amax(1, keepdim=True) / E4M3_MAX
            codes = _exact_codes(x, scale)
            if n == "exp_avg_sq":
                codes = torch.where((x > 0) & (codes == 0), torch.full_like(codes, E4M3_MIN), codes)
            out[n][one], out[n + "_scale"][few] = codes.view(-1), scale.view(-1)
    return out


def exact(case, seed):
    if case["op"] in ("forward", "train"):
        return _exact_ff(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(case, seed)
    total = math.sqrt(sum(float((t.double() * t.double()).sum()) for t in prepare(case, seed)["grad_flat"].split(1 << 26)))
    return {"norm": total, "scale": min(1.0, MAX_NORM / total)}
