"""AdamW on arrays refuses a clip factor that lies in a buffer the step writes."""
from __future__ import annotations

import pytest

import zengpu_b200 as zg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["weight", "exp_avg", "exp_avg_sq", "master", "exp_avg_scale",
                                   "exp_avg_sq_scale"])
def test_adamw_refuses_a_factor_it_would_write(device, pool, which):
    alloc = lambda n, dtype=zg.DType.F32: pool.alloc([n], dtype)  # noqa: E731
    n = 300 if "scale" in which else 2  # two blocks of 256, or the factor's own shape
    kind = zg.DType.Bf16 if which == "master" else zg.DType.F32
    codes = zg.DType.U8 if "scale" in which else zg.DType.F32
    arrays = {"weight": alloc(n, kind), "exp_avg": alloc(n, codes), "exp_avg_sq": alloc(n, codes),
              "master": alloc(n), "exp_avg_scale": alloc(2), "exp_avg_sq_scale": alloc(2)}
    grad = alloc(n)
    step = lambda factor: zg.Level1Kernels(device).adamw(  # noqa: E731
        device, [arrays["weight"]], [grad], [arrays["exp_avg"]], [arrays["exp_avg_sq"]], 1,
        master=[arrays["master"]] if which == "master" else None,
        scales=([arrays["exp_avg_scale"]], [arrays["exp_avg_sq_scale"]]) if "scale" in which else None,
        norm_scale=factor)
    with pytest.raises(zg.Dispatch, match="twice"):
        step(arrays[which])
    step(alloc(2))  # a buffer of its own
