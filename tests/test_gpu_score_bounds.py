"""GPU: score attention in f16 and bf16 within the bound of _score_bound.py, whose terms are those of
the exponentials, caps and roundings that the kernels have."""

import pytest
import torch

from fusionpass_b200 import fpkern
from tests._score_bound import reference
from tests._score_ref import close

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
SHAPES = [(2, 2, 2, 128, 128, 64), (1, 4, 2, 100, 100, 16), (1, 4, 1, 70, 300, 32), (2, 2, 1, 257, 513, 128),
          (1, 1, 1, 130, 4000, 128), (1, 160, 160, 300, 700, 128), (1, 2, 2, 640, 640, 64),
          (2, 8, 2, 1, 300, 128), (1, 16, 1, 1, 5000, 128), (2, 2, 1, 8, 1000, 16), (5, 4, 2, 2, 1500, 64)]


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kw", [{}, {"causal": True}, {"softcap": 5.0}, {"softcap": 50.0, "causal": True},
                                {"softcap": 1000.0}, {"slopes": 0.3, "causal": True}, {"slopes": 0.02, "softcap": 20.0},
                                {"causal": True, "window": 77, "prefix": 20}],
                         ids=["plain", "causal", "cap5", "cap50", "cap1000", "bias", "cap_bias", "window"])
def test_within_the_bound(dt, shape, kw):
    B, H, Hk, Sq, Sk, D = shape
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    # with a cap, scores as wide as it bites, and a few small ones
    wide = {None: 1.0, 1000.0: 300.0}.get(kw.get("softcap"), 8.0)
    q, k, v = (r(B, H, Sq, D) * wide).to(dt), r(B, Hk, Sk, D).to(dt), r(B, Hk, Sk, D).to(dt)
    kw = dict(kw)
    if "slopes" in kw:
        kw["slopes"] = torch.linspace(0.0, kw["slopes"], H, device="cuda")
    ref, bound = reference(q, k, v, D ** -0.5, **kw)
    close(fpkern.score_attention(q, k, v, D ** -0.5, **kw), ref, bound)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("Sq", [1, 200])
@pytest.mark.parametrize("D", [64, 128])
def test_two_keys_a_cap_apart(dt, Sq, D):
    """Two keys decide: a score's error moves the result by a quarter of it.  Scores over the whole cap."""
    g = torch.Generator(device="cuda").manual_seed(D + Sq)
    H, Sk = 64, 2
    v = torch.zeros(1, H, Sk, D, device="cuda", dtype=dt)
    v[:, :, 0] = 1.0
    for cap in (1.0, 30.0, 1000.0):
        q = torch.zeros(1, H, Sq, D, device="cuda")
        q[..., 0] = torch.randn(1, H, Sq, generator=g, device="cuda") * 2 * cap
        k = torch.zeros(1, H, Sk, D, device="cuda")
        k[:, :, 0, 0] = 1.0
        k[:, :, 1, 0] = 1.0 + 2.0 ** -5 * torch.randint(0, 9, (1, H), generator=g, device="cuda") / max(cap / 30, 1)
        q, k = q.to(dt), k.to(dt)
        ref, bound = reference(q, k, v, 1.0, softcap=cap)
        close(fpkern.score_attention(q, k, v, 1.0, softcap=cap), ref, bound)
