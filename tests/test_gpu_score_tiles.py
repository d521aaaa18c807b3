"""GPU: score attention where the two query tiles of one CTA (head dim 128, more than 128 queries)
have unequal key tiles, in calls large enough that no block's keys are split."""

import pytest
import torch

from fusionpass_b200 import fpkern
from tests._score_ref import close, reference, visible

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
# 24 x 8 heads x one block of two query tiles: more CTAs than SMs
B, H, HK, S, D = 24, 8, 2, 256, 128


def _inputs(dt, seed, sk=S):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").to(dt)  # noqa: E731
    return r(B, H, S, D), r(B, HK, sk, D), r(B, HK, sk, D)


def _empty(first):
    ids = torch.zeros(B, S, device="cuda", dtype=torch.int32)
    ids[:, :128] = -1 if first else 0
    ids[:, 128:] = 0 if first else -1
    return ids


def _lens(n):
    return torch.full((B,), n, device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("kw", [{"doc_ids": True}, {"doc_ids": False}, {"doc_ids": True, "causal": True},
                                {"causal": True, "kv_lens": 100}, {"causal": True, "kv_lens": 1},
                                {"causal": True, "kv_lens": 100, "softcap": 20.0},
                                {"causal": True, "kv_lens": 100, "window": 30}],
                         ids=["first_without_document", "last_without_document", "first_without_document_causal",
                              "short_cache", "one_key", "short_cache_cap", "short_cache_window"])
def test_one_query_tile_sees_no_key(dt, kw):
    """Its rows are zeros, whatever its queries hold: the staged zeros lie where its queries are loaded."""
    kw = dict(kw)
    if "doc_ids" in kw:
        kw["doc_ids"] = _empty(kw["doc_ids"])
    if "kv_lens" in kw:
        kw["kv_lens"] = _lens(kw["kv_lens"])
    q, k, v = _inputs(dt, 3)
    seen = visible(B, S, S, **{x: y for x, y in kw.items() if x != "softcap"})[0].any(-1)
    assert (~seen[:, :128]).all() or (~seen[:, 128:]).all()
    ref, bound = reference(q, k, v, D ** -0.5, **kw)
    none = ~seen[:, None, :, None].expand_as(q)
    for _ in range(20):
        out = torch.full_like(q, 7.0)
        fpkern.score_attention(q, k, v, D ** -0.5, out=out, **kw)
        assert out[none].eq(0).all()
        close(out, ref, bound)
    assert fpkern.poll_status() == 0
