"""GPU: RMS norms of many rows around the lengths where a row goes from ten elements a thread of
1024 to sixteen, and from the resident grid to a block a row."""

import pytest
import torch

from fusionpass_b200 import fpkern
from tests.test_gpu_rms_norm import EPS, _check_q, _check_y, _ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [5120, 5121, 7001, 10239, 10240, 10241, 12345, 16383, 16384])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
def test_long_rows_off_16_bytes(dt, n):
    """A base one element off; the elements before and behind the result stay as they were."""
    rows = 317
    g = torch.Generator(device="cuda").manual_seed(n)
    bufs = [torch.randn(rows * n + 2, generator=g, device="cuda").to(dt) for _ in range(2)]
    x, r = (b[1:1 + rows * n].view(rows, n) for b in bufs)
    w = (1 + 0.1 * torch.randn(n, generator=g, device="cuda")).to(dt)
    for adds in ([x], [x, r]):
        ref, _ = _ref(adds, w)
        buf = torch.full((rows * n + 2,), 7.0, device="cuda", dtype=dt)
        y, total = fpkern.add_rms_norm(adds, w, EPS, return_sum=True, out=buf[1:1 + rows * n].view(rows, n))
        _check_y(y, ref, adds, w, n)
        assert buf[0] == 7 and buf[-1] == 7
        assert torch.equal(total, sum(a.float() for a in adds).to(dt))
        q, scale, kept = fpkern.rms_norm_q8(adds, w, EPS, return_sum=True)
        _check_q(q, scale, ref, adds, n)
        assert torch.equal(kept, total)
    assert fpkern.poll_status() == 0
