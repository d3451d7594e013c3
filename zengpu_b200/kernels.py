"""Stream-level entry points on torch CUDA tensors (layer 3 of the C ABI).

Thin wrappers: shape / dtype / device checks in Python, then one call into
libzengpu_b200 with raw device pointers and torch's current CUDA stream.
torch only supplies device memory and streams here; every kernel that runs
is this library's own sm_100a code.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import functools
import threading
from typing import Sequence

import torch

from . import _lib as L
from .api import Activation, DType, GemmMode, check

ADAMW_BLOCK = 256  # elements that share a scale in 8-bit moments (ZG_ADAMW_BLOCK)

# One scratch tensor per (device, stream): GEMMs issued on different streams
# may overlap, and each stream reuses its own scratch in stream order.
_workspaces: dict[tuple[int, int], torch.Tensor] = {}

# A call queues several kernels that pass data through that scratch, and the interpreter
# lets other threads run meanwhile: a second call on the same stream must not queue its
# kernels between them.  (Reentrant: a finaliser may run a call of its own meanwhile.)
_queueing = threading.RLock()


def _stream(t: torch.Tensor) -> C.c_void_p:
    return C.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _f32_cuda(*ts: torch.Tensor) -> None:
    for t in ts:
        if t.dtype != torch.float32 or not t.is_cuda or not t.is_contiguous():
            raise ValueError("expected contiguous float32 CUDA tensors")


def add_f32(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """out = a + b, elementwise (bit-exact f32)."""
    _f32_cuda(a, b)
    if a.shape != b.shape:
        raise ValueError(f"add: shape mismatch {tuple(a.shape)} vs {tuple(b.shape)}")
    out = torch.empty_like(a) if out is None else out
    _f32_cuda(out)
    check(L.load().zg_add_f32(a.data_ptr(), b.data_ptr(), out.data_ptr(), a.numel(), _stream(a)))
    return out


def relu_f32(a: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """out = relu(a); pass out=a for the in-place form."""
    _f32_cuda(a)
    out = torch.empty_like(a) if out is None else out
    _f32_cuda(out)
    check(L.load().zg_relu_f32(a.data_ptr(), out.data_ptr(), a.numel(), _stream(a)))
    return out


def saxpy_f32(alpha: float, x: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    _f32_cuda(x, y)
    check(L.load().zg_saxpy_f32(float(alpha), x.data_ptr(), y.data_ptr(), x.numel(), _stream(x)))
    return y


def sscal_f32(alpha: float, x: torch.Tensor) -> torch.Tensor:
    _f32_cuda(x)
    check(L.load().zg_sscal_f32(float(alpha), x.data_ptr(), x.numel(), _stream(x)))
    return x


def workspace_bytes(mode: int, m: int, n: int, k: int) -> int:
    return int(L.load().zg_sgemm_workspace_bytes(int(mode), m, n, k))


def workspace_for(device: torch.device, nbytes: int) -> torch.Tensor | None:
    """Scratch tensor of the current stream on `device`, grown on demand
    (reused in stream order, so only GEMMs on that stream share it).  A capture gets
    memory of its own, which no other graph or stream shares: its graph may be
    replayed on any stream."""
    if nbytes == 0:
        return None
    idx = device.index if device.index is not None else torch.cuda.current_device()
    with _on(idx):
        if torch._C._cuda_isCurrentStreamCapturing():
            return torch.empty(nbytes, dtype=torch.uint8, device=device)
    key = (idx, torch.cuda.current_stream(idx).cuda_stream)
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        _workspaces[key] = ws
    return ws


def release_workspaces(device: torch.device | int | None = None) -> int:
    """Drops the cached GEMM scratch tensors (of one device, or of all) and
    returns how many were dropped.  The cache holds one tensor per (device,
    stream) that ever ran sgemm, each the size of that stream's largest GEMM,
    until this is called: code that creates short-lived streams should call it
    once those streams are done.  Dropping a tensor whose GEMM is still queued
    is safe: torch's caching allocator hands its memory out again only in the
    order of the stream it was allocated on (the stream it was cached for)."""
    if device is None:
        n = len(_workspaces)
        _workspaces.clear()
        return n
    idx = device if isinstance(device, int) else (
        device.index if device.index is not None else torch.cuda.current_device())
    keys = [key for key in _workspaces if key[0] == idx]
    for key in keys:
        del _workspaces[key]
    return len(keys)


def sgemm(a: torch.Tensor, b: torch.Tensor, mode: int = GemmMode.TF32X3, alpha: float = 1.0,
          bias: torch.Tensor | None = None, relu: bool = False,
          out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """C = epilogue(alpha * a @ b) for row-major f32 a [m,k], b [k,n]."""
    _f32_cuda(a, b)
    if a.dim() != 2 or b.dim() != 2 or a.shape[1] != b.shape[0]:
        raise ValueError(f"sgemm: bad shapes {tuple(a.shape)} @ {tuple(b.shape)}")
    m, k = a.shape
    n = b.shape[1]
    if bias is not None:
        _f32_cuda(bias)
        if bias.numel() != n:
            raise ValueError("sgemm: bias must have n elements")
    out = torch.empty((m, n), dtype=torch.float32, device=a.device) if out is None else out
    _f32_cuda(out)
    need = workspace_bytes(mode, m, n, k)
    with _queueing:
        ws = workspace if workspace is not None else workspace_for(a.device, need)
        ws_ptr = ws.data_ptr() if ws is not None else None
        ws_len = ws.numel() if ws is not None else 0
        rc = L.load().zg_sgemm_f32(int(mode), m, n, k, float(alpha), a.data_ptr(), b.data_ptr(),
                                   out.data_ptr(), bias.data_ptr() if bias is not None else None,
                                   1 if relu else 0, ws_ptr, ws_len, _stream(a))
    check(rc)
    return out


def fill_uniform(t: torch.Tensor, seed: int, lo: float = -1.0, hi: float = 1.0) -> torch.Tensor:
    _f32_cuda(t)
    check(L.load().zg_fill_uniform_f32(t.data_ptr(), t.numel(), int(seed), float(lo), float(hi),
                                       _stream(t)))
    return t


def fill_normal(t: torch.Tensor, seed: int) -> torch.Tensor:
    _f32_cuda(t)
    check(L.load().zg_fill_normal_f32(t.data_ptr(), t.numel(), int(seed), _stream(t)))
    return t


def kernel_status() -> int:
    """Reads and clears the device status word (0 = every bounded wait finished)."""
    code = C.c_uint32(0)
    check(L.load().zg_kernel_status(C.byref(code)))
    return int(code.value)


# ---- packed operands (zg_sgemm_pack_*, zg_sgemm_packed) ----------------------------
class Packed:
    """An operand packed for one GEMM mode: the planes its kernel reads."""

    def __init__(self, mode: int, operand: int, outer: int, k: int, buf: torch.Tensor):
        self.mode, self.operand, self.outer, self.k, self.buf = int(mode), operand, outer, k, buf


def pack_bytes(mode: int, operand: int, outer: int, k: int) -> int:
    return int(L.load().zg_sgemm_pack_bytes(int(mode), operand, outer, k))


def _pack_buffer(nbytes: int, device, out: torch.Tensor | None) -> torch.Tensor:
    if out is not None and out.numel() >= nbytes and out.data_ptr() % 256 == 0:
        return out
    return torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)


def _pitch(t: torch.Tensor) -> int:
    if t.dim() != 2 or t.stride(1) != 1:
        raise ValueError("expected a 2-D float32 CUDA tensor with unit column stride")
    return t.stride(0)


def pack_a(a: torch.Tensor, mode: int = GemmMode.TF32X3, out: torch.Tensor | None = None) -> Packed:
    """Packs A [m, k] (any row pitch) for `mode`."""
    if a.dtype != torch.float32 or not a.is_cuda:
        raise ValueError("pack_a: float32 CUDA tensor expected")
    m, k = a.shape
    buf = _pack_buffer(pack_bytes(mode, 0, m, k), a.device, out)
    check(L.load().zg_sgemm_pack_a(int(mode), m, k, a.data_ptr(), _pitch(a), buf.data_ptr(),
                                   buf.numel(), _stream(a)))
    return Packed(mode, 0, m, k, buf)


def pack_b(b: torch.Tensor, mode: int = GemmMode.TF32X3, out: torch.Tensor | None = None) -> Packed:
    """Packs B [k, n] (any row pitch) for `mode`."""
    if b.dtype != torch.float32 or not b.is_cuda:
        raise ValueError("pack_b: float32 CUDA tensor expected")
    k, n = b.shape
    buf = _pack_buffer(pack_bytes(mode, 1, n, k), b.device, out)
    check(L.load().zg_sgemm_pack_b(int(mode), k, n, b.data_ptr(), _pitch(b), buf.data_ptr(),
                                   buf.numel(), _stream(b)))
    return Packed(mode, 1, n, k, buf)


def sgemm_packed(pa: Packed, pb: Packed, c: torch.Tensor | None = None, alpha: float = 1.0,
                 bias: torch.Tensor | None = None, relu: bool = False) -> torch.Tensor:
    """C = epilogue(alpha * A @ B) from packed operands; `c` may be a column
    panel view of a larger row-major matrix (row pitch = c.stride(0))."""
    if pa.mode != pb.mode or pa.k != pb.k or pa.operand != 0 or pb.operand != 1:
        raise ValueError("sgemm_packed: operands packed for different GEMMs")
    m, n, k = pa.outer, pb.outer, pa.k
    if c is None:
        c = torch.empty((m, n), dtype=torch.float32, device=pa.buf.device)
    if tuple(c.shape) != (m, n) or c.dtype != torch.float32:
        raise ValueError(f"sgemm_packed: C must be float32 [{m}, {n}]")
    if bias is not None:
        _f32_cuda(bias)
    check(L.load().zg_sgemm_packed(pa.mode, m, n, k, float(alpha), pa.buf.data_ptr(),
                                   pb.buf.data_ptr(), c.data_ptr(), _pitch(c),
                                   bias.data_ptr() if bias is not None else None,
                                   1 if relu else 0, _stream(c)))
    return c


# ---- gated feed-forward block (zg_gated_ff, zg_gated_ff_backward) ----------------------
_FLOATS = {torch.float32: DType.F32, torch.float16: DType.F16, torch.bfloat16: DType.Bf16}


def _on(index: int):
    """Makes device `index` the current one for a call (free when it already is)."""
    return contextlib.nullcontext() if index == torch._C._cuda_getDevice() \
        else torch.cuda.device(index)


def _raw_stream(index: int) -> int:
    """_stream without the Stream object around it: a call of a few microseconds notices."""
    return torch._C._cuda_getCurrentRawStream(index)


def _scratch(index: int, stream: int, nbytes: int) -> torch.Tensor | None:
    """workspace_for of a device, the current one, and a stream known by number."""
    if nbytes == 0:
        return None
    ws = _workspaces.get((index, stream))
    if ws is not None and ws.numel() >= nbytes and not torch._C._cuda_isCurrentStreamCapturing():
        return ws
    return workspace_for(torch.device("cuda", index), nbytes)


def _ff_operand(name: str, t: torch.Tensor, shape: tuple[int, ...],
                like: torch.Tensor) -> torch.Tensor:
    if t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {shape}")
    if t.dtype is not like.dtype or t.device != like.device or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous {like.dtype} tensor on {like.device}")
    # the kernels' copies start on 16-byte boundaries; a view that does not is copied
    return t if t.data_ptr() % 16 == 0 else t.detach().clone()


def _ff_output(name: str, t: torch.Tensor | None, shape: tuple[int, ...],
               like: torch.Tensor, dtype: torch.dtype | None = None) -> torch.Tensor:
    if t is None:
        return like.new_empty(shape) if dtype is None else like.new_empty(shape, dtype=dtype)
    dtype = dtype or like.dtype
    if t.dtype != dtype or t.device != like.device or not t.is_contiguous() or t.shape != shape:
        raise ValueError(f"{name}: expected a contiguous {dtype} tensor of shape {shape}")
    return t


def _apart(outs: dict[str, torch.Tensor | None], ins: dict[str, torch.Tensor]) -> None:
    """Refuses given outputs that overlap an input, or each other: kernels read the one
    while they write the other."""
    def span(t):
        return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()
    given = [(name, t, *span(t)) for name, t in outs.items() if t is not None and t.numel()]
    others = given + [(name, t, *span(t)) for name, t in ins.items()]
    for i, (name, t, a, b) in enumerate(given):
        for other, o, c, d in others[i + 1:]:
            if a < d and c < b and t.device == o.device:
                raise ValueError(f"{name}: overlaps {other}")


def _ff_sizes(x: torch.Tensor, w_gate: torch.Tensor, w_down: torch.Tensor) -> tuple[int, ...]:
    if not x.is_cuda or x.dtype not in _FLOATS:
        raise ValueError("gated_ff: expected f32, bf16 or f16 CUDA tensors")
    if x.dim() != 2 or w_gate.dim() != 2 or w_down.dim() != 2:
        raise ValueError("gated_ff: expected 2-D tensors")
    sizes = (*x.shape, w_gate.shape[1], w_down.shape[1])
    if max(sizes) > 1 << 28:
        raise ValueError(f"gated_ff: sizes {sizes} exceed 2^28")
    return sizes


def _ff_ready(index: int, dtype: torch.dtype, pairs) -> bool:
    """Whether each (tensor, shape) is as the kernels take it, on the current device."""
    if index != torch._C._cuda_getDevice():
        return False
    for t, shape in pairs:
        if t.dtype is not dtype or t.shape != shape or t.get_device() != index or \
                not t.is_contiguous() or t.data_ptr() & 15:
            return False
    return True


@functools.lru_cache(maxsize=1024)
def _ff_workspace_bytes(dtype: int, mode: int, m: int, k: int, f: int, d: int,
                        backward: int) -> int:
    return int(L.load().zg_gated_ff_workspace_bytes(dtype, mode, m, k, f, d, backward))


def gated_ff(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
             act: int = Activation.SILU, mode: int = GemmMode.TF32X3, save: bool = False,
             out: torch.Tensor | None = None):
    """y = (act(x @ w_gate) * (x @ w_up)) @ w_down for contiguous x [m, k], w_gate
    and w_up [k, f], w_down [f, d] of one dtype: f32 (in `mode`, as sgemm), bf16 or
    f16 (f32 sums; the inner product is rounded once to the dtype).  save=True
    returns (y, saved), `saved` being what gated_ff_backward needs: the two inner
    products before the activation, f32 [m, f] each.  `out` overlaps no input."""
    m, k, f, d = _ff_sizes(x, w_gate, w_down)
    index = x.get_device()
    if out is not None:
        _apart({"out": out}, {"x": x, "w_gate": w_gate, "w_up": w_up, "w_down": w_down})
    if not _ff_ready(index, x.dtype, ((x, (m, k)), (w_gate, (k, f)), (w_up, (k, f)),
                                      (w_down, (f, d)))):
        with _on(index):
            x = _ff_operand("x", x, (m, k), x)
            w_gate = _ff_operand("w_gate", w_gate, (k, f), x)
            w_up = _ff_operand("w_up", w_up, (k, f), x)
            w_down = _ff_operand("w_down", w_down, (f, d), x)
            return _gated_ff(index, m, k, f, d, x, w_gate, w_up, w_down, act, mode, save, out)
    return _gated_ff(index, m, k, f, d, x, w_gate, w_up, w_down, act, mode, save, out)


def _gated_ff(index, m, k, f, d, x, w_gate, w_up, w_down, act, mode, save, out):
    y = _ff_output("out", out, (m, d), x)
    saved = (x.new_empty((m, f), dtype=torch.float32),
             x.new_empty((m, f), dtype=torch.float32)) if save else None
    dt, stream, mode = _FLOATS[x.dtype].value, _raw_stream(index), int(mode)
    need = _ff_workspace_bytes(dt, mode, m, k, f, d, 0)
    with _queueing:
        ws = _scratch(index, stream, need)
        rc = L.load().zg_gated_ff(
            dt, mode, int(act), m, k, f, d, x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(),
            w_down.data_ptr(), y.data_ptr(), saved[0].data_ptr() if save else None,
            saved[1].data_ptr() if save else None, ws.data_ptr() if ws is not None else None,
            need, stream)
    check(rc)
    return (y, saved) if save else y


def gated_ff_backward(dy: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor,
                      w_up: torch.Tensor, w_down: torch.Tensor,
                      saved: tuple[torch.Tensor, torch.Tensor], act: int = Activation.SILU,
                      mode: int = GemmMode.TF32X3,
                      out: Sequence[torch.Tensor | None] = (None, None, None, None)):
    """(dx, dw_gate, dw_up, dw_down) of gated_ff for dy, the gradient of its y;
    `saved` as gated_ff(..., save=True) gave it for the same x and weights.  `out`
    takes tensors to write them to, which overlap neither an input nor one another."""
    m, k, f, d = _ff_sizes(x, w_gate, w_down)
    index, act, mode = x.get_device(), int(act), int(mode)
    if len(saved) != 2 or any(t is None for t in saved):
        raise ValueError("gated_ff_backward: saved has two tensors")
    if len(out) != 4:
        raise ValueError("gated_ff_backward: out has four places")
    if any(t is not None for t in out):
        _apart(dict(zip(("dx", "dw_gate", "dw_up", "dw_down"), out)),
               {"dy": dy, "x": x, "w_gate": w_gate, "w_up": w_up, "w_down": w_down,
                "saved[0]": saved[0], "saved[1]": saved[1]})
    with _on(index):
        x = _ff_operand("x", x, (m, k), x)
        dy = _ff_operand("dy", dy, (m, d), x)
        w_gate = _ff_operand("w_gate", w_gate, (k, f), x)
        w_up = _ff_operand("w_up", w_up, (k, f), x)
        w_down = _ff_operand("w_down", w_down, (f, d), x)
        pre = [_ff_output("saved", t, (m, f), x, torch.float32) for t in saved]
        pre = [t if t.data_ptr() % 16 == 0 else t.detach().clone() for t in pre]
        got = (_ff_output("dx", out[0], (m, k), x), _ff_output("dw_gate", out[1], (k, f), x),
               _ff_output("dw_up", out[2], (k, f), x), _ff_output("dw_down", out[3], (f, d), x))
        dt, stream = _FLOATS[x.dtype].value, _raw_stream(index)
        need = _ff_workspace_bytes(dt, mode, m, k, f, d, 1)
        with _queueing:
            ws = _scratch(index, stream, need)
            rc = L.load().zg_gated_ff_backward(
                dt, mode, act, m, k, f, d, dy.data_ptr(), x.data_ptr(), w_gate.data_ptr(),
                w_up.data_ptr(), w_down.data_ptr(), pre[0].data_ptr(), pre[1].data_ptr(),
                *[t.data_ptr() for t in got], ws.data_ptr() if ws is not None else None, need,
                stream)
        check(rc)
    return got


# ---- AdamW over many tensors, gradient norm (zg_adamw, zg_grad_norm) -------------------
def _same(name: str, tensors: Sequence[torch.Tensor], like: Sequence[int],
          device: torch.device, dtypes: Sequence[torch.dtype]) -> None:
    """Checks a list of contiguous CUDA tensors: one dtype out of `dtypes`, `like` elements each."""
    if len(tensors) != len(like):
        raise ValueError(f"{name}: {len(tensors)} tensors, expected {len(like)}")
    for t, n in zip(tensors, like):
        if t.device != device or not t.is_contiguous():
            raise ValueError(f"{name}: expected contiguous tensors on {device}")
        if t.dtype not in dtypes or t.dtype != tensors[0].dtype:
            raise ValueError(f"{name}: unexpected dtype {t.dtype}")
        if t.numel() != n:
            raise ValueError(f"{name}: {t.numel()} elements, expected {n}")


def _device_scalar(name: str, t: torch.Tensor, dtype: torch.dtype,
                   device: torch.device) -> int:
    if t.dtype != dtype or t.numel() != 1 or t.device != device:
        raise ValueError(f"{name}: expected one {dtype} on {device}")
    return t.data_ptr()


class AdamW:
    """AdamW over many tensors, one launch a step (zg_adamw): in place on the
    weights, their moments and, for 16-bit weights, their f32 `master` copies.

    params: f32, bf16 or f16 CUDA tensors of one dtype; grads: as many, of one
    dtype, the buffers every step reads; state_bits: 32 (f32 moments) or 8 (e4m3
    codes of m and of sqrt(v), with an f32 scale for each 256 elements).
    `state` takes the moments a program already has, as lists by name; by
    default they start at zero.  All tensors are contiguous and none overlaps
    another.  The object keeps them alive; a step runs on the current stream."""

    def __init__(self, params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor],
                 state_bits: int = 32, master: Sequence[torch.Tensor] | None = None,
                 state: dict[str, Sequence[torch.Tensor]] | None = None):
        if not params:
            raise ValueError("AdamW: no tensors")
        if state_bits not in (32, 8):
            raise ValueError(f"AdamW: state_bits is 32 or 8, got {state_bits}")
        device = params[0].device
        if device.type != "cuda":
            raise ValueError("AdamW: expected CUDA tensors")
        sizes = [p.numel() for p in params]
        blocks = [-(-n // ADAMW_BLOCK) for n in sizes]
        _same("AdamW params", params, sizes, device, tuple(_FLOATS))
        _same("AdamW grads", grads, sizes, device, tuple(_FLOATS))
        if master is not None:
            if params[0].dtype == torch.float32:
                raise ValueError("AdamW: f32 weights take no master")
            _same("AdamW master", master, sizes, device, (torch.float32,))
        moments = {"exp_avg": sizes, "exp_avg_sq": sizes}
        if state_bits == 8:
            moments |= {"exp_avg_scale": blocks, "exp_avg_sq_scale": blocks}
        if state is not None and set(state) != set(moments):
            raise ValueError(f"AdamW: state has {sorted(state)}, expected {sorted(moments)}")
        self.state: dict[str, list[torch.Tensor]] = {}
        for name, counts in moments.items():
            codes = state_bits == 8 and not name.endswith("scale")
            dtype = torch.float8_e4m3fn if codes else torch.float32
            if state is None:
                self.state[name] = [torch.zeros(n, dtype=torch.uint8 if codes else dtype,
                                                device=device).view(dtype) for n in counts]
            else:
                _same(f"AdamW {name}", state[name], counts, device, (dtype,))
                self.state[name] = list(state[name])
        self.params, self.grads, self.state_bits = list(params), list(grads), state_bits
        self.master = list(master) if master is not None else None
        written = [self.params, self.master or [], *self.state.values()]
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), kind)
                       for kind, ts in ((1, sum(written, [])), (0, self.grads))
                       for t in ts if t.numel())
        end, kind = 0, 0
        for a, b, k in spans:
            if a < end and (k or kind):  # two gradients may be the same memory
                raise ValueError("AdamW: tensors overlap")
            end, kind = (b, k) if b >= end else (end, kind | k)
        self._device = device
        self._types = (_FLOATS[params[0].dtype].value, _FLOATS[grads[0].dtype].value)
        self._table = (L.AdamWTensor * len(params))()
        for i, row in enumerate(self._table):
            row.param, row.grad, row.n = params[i].data_ptr(), grads[i].data_ptr(), sizes[i]
            row.master = self.master[i].data_ptr() if self.master else None
            for name, ts in self.state.items():
                setattr(row, name, ts[i].data_ptr())

    def step(self, step: int | torch.Tensor, lr: float | torch.Tensor = 1e-3, beta1: float = 0.9,
             beta2: float = 0.999, eps: float = 1e-8, weight_decay: float = 0.01,
             grad_scale: torch.Tensor | None = None) -> None:
        """Step number `step` (from 1).  `step` (int64) and `lr` (float32) may be
        device scalars, which a captured step reads anew at each replay.
        grad_scale: a float32 device scalar the gradients are multiplied by, as
        GradNorm gives it; when it is not finite the step changes nothing."""
        device = self._device
        step_dev = lr_dev = scale_dev = None
        if isinstance(step, torch.Tensor):
            step_dev, step = _device_scalar("AdamW step", step, torch.int64, device), 0
        if isinstance(lr, torch.Tensor):
            lr_dev, lr = _device_scalar("AdamW lr", lr, torch.float32, device), 0.0
        if grad_scale is not None:
            scale_dev = _device_scalar("AdamW grad_scale", grad_scale, torch.float32, device)
        hyper = L.AdamWHyper(lr, beta1, beta2, eps, weight_decay, step)
        with _on(device.index):
            check(L.load().zg_adamw(*self._types, self.state_bits, len(self._table), self._table,
                                    hyper, step_dev, lr_dev, scale_dev, _raw_stream(device.index)))


class GradNorm:
    """The 2-norm over many gradients (zg_grad_norm), and the factor that clips
    them.  grads: contiguous CUDA tensors of one dtype (f32, bf16 or f16), read
    anew by every call."""

    def __init__(self, grads: Sequence[torch.Tensor]):
        if not grads or grads[0].device.type != "cuda":
            raise ValueError("GradNorm: expected CUDA tensors")
        self._device = grads[0].device
        _same("GradNorm", grads, [g.numel() for g in grads], self._device, tuple(_FLOATS))
        self.grads = list(grads)
        self._type = _FLOATS[grads[0].dtype].value
        self._ptrs = (C.c_void_p * len(grads))(*[g.data_ptr() for g in grads])
        self._sizes = (C.c_uint64 * len(grads))(*[g.numel() for g in grads])
        self._ws_bytes = int(L.load().zg_grad_norm_workspace_bytes(len(grads)))

    def clip_scale(self, max_norm: float) -> torch.Tensor:
        """[norm, min(1, max_norm / norm)] as two f32 on the device; the factor is
        NaN when the norm is not finite.  out[1:] is AdamW.step's grad_scale."""
        index = self._device.index
        with _on(index):
            stream = _raw_stream(index)
            out = self.grads[0].new_empty(2, dtype=torch.float32)
            with _queueing:
                ws = _scratch(index, stream, self._ws_bytes)
                rc = L.load().zg_grad_norm(self._type, len(self._sizes), self._ptrs, self._sizes,
                                           max_norm, out.data_ptr(), ws.data_ptr(),
                                           self._ws_bytes, stream)
            check(rc)
        return out
