"""Calls from several threads: those that pass data through a stream's scratch memory
queue their kernels one call after the other (a fake library stands in, so no GPU is
needed); on the GPU, threads that share a stream get the bits of a call alone."""
from __future__ import annotations

import threading
import time

import pytest
import torch

from zengpu_b200 import kernels as K


class Library:
    """Stands in for the library: notes calls that overlap."""

    def __init__(self):
        self.inside, self.overlaps, self.calls = 0, 0, []

    def __getattr__(self, name):
        def call(*args):
            self.inside += 1
            self.overlaps += self.inside > 1
            self.calls.append(name)
            time.sleep(0.02)  # lets the other threads run, as a foreign call does
            self.inside -= 1
            return 0
        return call


def test_calls_that_share_scratch_do_not_interleave(monkeypatch):
    lib = Library()
    monkeypatch.setattr(K.L, "load", lambda: lib)
    monkeypatch.setattr(K, "_scratch", lambda index, stream, nbytes: torch.empty(16))
    monkeypatch.setattr(K, "_ff_workspace_bytes", lambda *a: 16)
    monkeypatch.setattr(K, "workspace_bytes", lambda *a: 16)
    monkeypatch.setattr(K, "workspace_for", lambda *a: torch.empty(16))
    monkeypatch.setattr(K, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(K, "_stream", lambda t: None)
    monkeypatch.setattr(K, "_on", lambda index: K.contextlib.nullcontext())
    monkeypatch.setattr(K, "_f32_cuda", lambda *ts: None)
    monkeypatch.setattr(K, "_ff_sizes", lambda x, wg, wd: (*x.shape, wg.shape[1], wd.shape[1]))
    x, wg, wd, dy = torch.zeros(2, 4), torch.zeros(4, 6), torch.zeros(6, 5), torch.zeros(2, 5)
    saved = torch.zeros(2, 6), torch.zeros(2, 6)
    norm = object.__new__(K.GradNorm)
    norm._device, norm.grads, norm._type, norm._ws_bytes = torch.device("cpu", 0), [x], 0, 16
    norm._ptrs, norm._sizes = (), ()
    calls = [lambda: K._gated_ff(0, 2, 4, 6, 5, x, wg, wg, wd, 0, 1, False, None),
             lambda: K.gated_ff_backward(dy, x, wg, wg, wd, saved), lambda: norm.clip_scale(1.0),
             lambda: K.sgemm(x, wg)]
    threads = [threading.Thread(target=c) for c in calls for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert sorted(set(lib.calls)) == ["zg_gated_ff", "zg_gated_ff_backward", "zg_grad_norm",
                                      "zg_sgemm_f32"] and len(lib.calls) == 12
    assert lib.overlaps == 0


@pytest.mark.gpu
def test_threads_on_one_stream():
    gen = torch.Generator(device="cuda").manual_seed(0)
    def normal(*shape, kind=torch.bfloat16):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(0.1).to(kind)
    work = []
    for m, k, f, d, kind in ((40, 256, 520, 264, torch.bfloat16), (200, 256, 1032, 264, torch.float16),
                             (100, 130, 515, 77, torch.float32)):
        x, wg, wu, wd, dy = (normal(*s, kind=kind) for s in ((m, k), (k, f), (k, f), (f, d), (m, d)))
        plan = K.GradNorm([wg, wu])
        def one(x=x, wg=wg, wu=wu, wd=wd, dy=dy, plan=plan):
            y, saved = K.gated_ff(x, wg, wu, wd, save=True)
            return y, *saved, *K.gated_ff_backward(dy, x, wg, wu, wd, saved), plan.clip_scale(1.0)
        work.append((one, one()))
    torch.cuda.synchronize()
    wrong = []
    def run(one, want):
        for _ in range(50):
            got = one()
            torch.cuda.current_stream().synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want)):
                wrong.append(1)
    threads = [threading.Thread(target=run, args=w) for w in work * 2]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and K.kernel_status() == 0
