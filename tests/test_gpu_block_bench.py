"""GPU: benchmark() on a verified model of the quantised block."""

import pytest
import torch

from fusionpass_b200 import benchmark, compile_model
from tests.block_models import QuantHead

pytestmark = pytest.mark.gpu


def test_benchmark_of_a_verified_head():
    m = QuantHead().eval().to("cuda")
    xs = tuple(torch.randn(70, 96, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i)) for i in range(2))
    # off by steps of single activations: 5 / 127 of a normalised row at most, times a weight
    kw = {"atol": 5 / 127 * 4 * 96 ** -0.5, "rtol": 1e-3, "extensions": True}
    c, plain = compile_model(m, xs, fuse=True, **kw), compile_model(m, xs, fuse=False, **kw)
    r = benchmark(m, c, xs, unfused=plain, warmup=3, iters=10)
    assert r.fused_ms > 0 and r.est_bytes_fused < r.est_bytes_unfused and r.fused_launches == 1
