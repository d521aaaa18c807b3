"""GPU: 8-bit caches of layouts that the kernels do not read where they are."""

import pytest
import torch

from fusionpass_b200 import fpkern

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["off", "columns", "pitch", "expanded"])
def test_read_takes_any_layout(dt, layout):
    """A base or rows off 16 bytes, head dims that are no unit stride, one cache for all sequences."""
    B, Hk, N, D = 3, 2, 37, 32
    g = torch.Generator(device="cuda").manual_seed(9)
    plain = [torch.randint(-127, 128, (B, Hk, N, D), generator=g, device="cuda").to(torch.int8) for _ in range(2)]
    ks, vs = (torch.rand(B, Hk, N, generator=g, device="cuda") for _ in range(2))
    if layout == "expanded":
        plain = [t[:1].expand(B, Hk, N, D) for t in plain]
        odd = plain
    elif layout == "columns":
        odd = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in plain]
    else:
        wide = D + (16 if layout == "off" else 5)
        odd = [torch.zeros(B, Hk, N, wide, dtype=torch.int8, device="cuda")[..., (3 if layout == "off" else 0):][..., :D] for _ in plain]
        for a, b in zip(odd, plain):
            a.copy_(b)
    lens = torch.tensor([N, 5, 0], dtype=torch.int32, device="cuda")
    for kv_lens in (None, lens):
        held = (torch.arange(N, device="cuda") < (lens if kv_lens is not None else lens[:1].expand(B))[:, None])[:, None, :, None]
        for got, c, s in zip(fpkern.cache_read_q8(*odd, ks, vs, dtype=dt, kv_lens=kv_lens), plain, (ks, vs)):
            assert got.is_contiguous() and torch.equal(got, torch.where(held, c.float() * s.unsqueeze(-1), 0.0).to(dt))
    x = torch.randn(B, Hk, 4, D, device="cuda", dtype=dt)
    before = [t.clone() for t in odd]
    with pytest.raises(ValueError):
        fpkern.cache_write_q8(x, x, *odd, ks, vs, lens)
    assert all(torch.equal(a, b) for a, b in zip(odd, before))
