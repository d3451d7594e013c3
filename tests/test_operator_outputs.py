"""Given outputs of the gated block: one that overlaps an input, or another output, is
refused before anything runs.  Tensors on the CPU stand in where the call gets no further."""
from __future__ import annotations

import pytest
import torch

from zengpu_b200 import kernels as K

M, SIZE = 4, 8  # all matrices square but for the rows, so that any may be taken for another


def tensors(device="cpu"):
    make = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=device)  # noqa: E731
    ins = {"x": make(M, SIZE), "w_gate": make(SIZE, SIZE), "w_up": make(SIZE, SIZE),
           "w_down": make(SIZE, SIZE)}
    saved = tuple(torch.zeros(M, SIZE, device=device) for _ in range(2))
    return ins, make(M, SIZE), saved


@pytest.fixture
def sizes(monkeypatch):
    """The checks before the overlap take CPU tensors."""
    monkeypatch.setattr(K, "_ff_sizes", lambda x, wg, wd: (M, SIZE, SIZE, SIZE))


@pytest.mark.parametrize("name", ["x", "w_gate", "w_up", "w_down"])
def test_forward_output_over_an_input(name, sizes):
    ins, _, _ = tensors()
    with pytest.raises(ValueError, match=f"out: overlaps {name}"):
        K.gated_ff(*ins.values(), out=ins[name].view(-1)[-M * SIZE:].view(M, SIZE))


@pytest.mark.parametrize("name", ["dy", "x", "w_gate", "w_up", "w_down", "saved[0]", "saved[1]"])
@pytest.mark.parametrize("place", range(4))
def test_gradient_over_an_input(place, name, sizes):
    ins, dy, saved = tensors()
    taken = (ins | {"dy": dy, "saved[0]": saved[0], "saved[1]": saved[1]})[name].view(-1)
    out = [None] * 4
    out[place] = taken[-1:]  # a single element is enough
    with pytest.raises(ValueError, match="overlaps " + name.replace("[", r"\[").replace("]", r"\]")):
        K.gated_ff_backward(dy, *ins.values(), saved, out=out)


@pytest.mark.parametrize("a,b", [(a, b) for a in range(4) for b in range(a)])
def test_gradients_over_one_another(a, b, sizes):
    ins, dy, saved = tensors()
    flat = torch.zeros(100, dtype=torch.bfloat16)
    out = [None] * 4
    out[a], out[b] = flat[:40], flat[39:]
    with pytest.raises(ValueError, match="overlaps"):
        K.gated_ff_backward(dy, *ins.values(), saved, out=out)


@pytest.mark.gpu
def test_neighbours_in_one_buffer_are_taken():
    """Outputs side by side in one buffer, and beside their inputs, do not overlap."""
    flat = torch.randn(8 * 64 * 64, device="cuda").to(torch.bfloat16)
    x, wg, wu, wd, *out = (flat[i * 4096:(i + 1) * 4096].view(64, 64) for i in range(8))
    dy = torch.randn(64, 64, device="cuda").to(torch.bfloat16)
    y, saved = K.gated_ff(x, wg, wu, wd, save=True)
    want = K.gated_ff_backward(dy, x, wg, wu, wd, saved)
    got = K.gated_ff_backward(dy, x, wg, wu, wd, saved, out=out)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    given = K.gated_ff(x, wg, wu, wd, out=out[0])
    assert given is out[0] and torch.equal(given, y)
    none = flat[:0].view(0, 64)
    assert K.gated_ff(none, wg, wu, wd, out=none).shape == (0, 64)
