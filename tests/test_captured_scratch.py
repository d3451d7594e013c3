"""Scratch memory of captured calls: a graph has its own, since it may be replayed on any
stream, beside eager calls and other graphs."""
from __future__ import annotations

import types

import pytest
import torch

from zengpu_b200 import GemmMode, kernels as K


def test_a_capture_neither_takes_nor_leaves_cached_scratch(monkeypatch):
    capturing = [False]
    monkeypatch.setattr(K, "_workspaces", {})
    monkeypatch.setattr(K, "_on", lambda index: K.contextlib.nullcontext())
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: capturing[0], raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda idx: types.SimpleNamespace(cuda_stream=7))
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, device=None, **kw: empty(*a, **kw))
    device = torch.device("cuda", 0)
    capturing[0] = True
    first, second = K.workspace_for(device, 64), K._scratch(0, 7, 64)
    assert first is not second and not K._workspaces
    capturing[0] = False
    eager = K.workspace_for(device, 64)
    assert K.workspace_for(device, 32) is eager and K._scratch(0, 7, 64) is eager
    assert K._scratch(0, 7, 128) is K.workspace_for(device, 128) is not eager
    capturing[0] = True
    assert K.workspace_for(device, 32) is not K._workspaces[(0, 7)] is not K._scratch(0, 7, 32)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [m for m in GemmMode if m != GemmMode.SIMT_FP32],
                         ids=lambda m: m.name)
def test_graphs_on_two_streams(mode):
    """Two graphs captured on one stream, replayed on two beside eager calls on the stream
    of the capture, give the bits of a call alone."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    pairs = [[torch.randn(*s, generator=gen, device="cuda") for s in ((700, 900), (900, 1100))]
             for _ in range(3)]
    want = [K.sgemm(a, b, mode=mode) for a, b in pairs]
    capture, *streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    graphs, held = [], []
    for a, b in pairs[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=capture):
            held.append(K.sgemm(a, b, mode=mode))
        graphs.append(graph)
    outs = []
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(capture):
            outs.append(K.sgemm(*pairs[2], mode=mode))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(held, want))
    assert all(torch.equal(x, want[2]) for x in outs) and K.kernel_status() == 0
