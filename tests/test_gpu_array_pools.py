"""A pool of another device object: the block and the gradient norm on arrays refuse it.
Handles are numbers within a device, so its array could name a buffer that is in use."""
from __future__ import annotations

import pytest

import zengpu_b200 as zg

pytestmark = pytest.mark.gpu


def test_pool_of_another_device_is_refused(device, pool):
    gemm, level1 = zg.GemmKernel(device), zg.Level1Kernels(device)
    alloc = lambda *s: pool.alloc(list(s), zg.DType.F32)  # noqa: E731
    x, wg, wu, wd, dy = alloc(4, 8), alloc(8, 16), alloc(8, 16), alloc(16, 8), alloc(4, 8)
    saved = alloc(4, 16), alloc(4, 16)
    other = zg.CudaDevice(0)
    foreign = zg.BufferPool(other)
    try:
        with pytest.raises(zg.Dispatch, match="another device"):
            gemm.gated_ff(device, foreign, x, wg, wu, wd)
        with pytest.raises(zg.Dispatch, match="another device"):
            gemm.gated_ff_backward(device, foreign, dy, x, wg, wu, wd, saved)
        with pytest.raises(zg.Dispatch, match="another device"):
            level1.grad_norm(device, foreign, [wg, wu], 1.0)
    finally:
        foreign.close()
        other.close()
    assert gemm.gated_ff(device, pool, x, wg, wu, wd).shape == [4, 8]
    assert level1.grad_norm(device, pool, [wg, wu], 1.0).shape == [2]
