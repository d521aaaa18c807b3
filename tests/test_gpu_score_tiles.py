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


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("n, kw", [(250, {"causal": True}), (200, {"causal": True, "window": 90}),
                                   (129, {"causal": True, "softcap": 20.0}), (250, {"doc_ids": True}),
                                   (S, {"causal": True})], ids=["causal", "window", "cap", "documents", "whole_cache"])
def test_values_that_are_not_finite_in_a_tile_of_the_other_rows(dt, value, n, kw):
    """NaN or infinities behind the keys, in the last key tile, which only the second query tile
    walks: the first one ends while they are noted.  One value that rows of both see is theirs."""
    kw = {**kw, "kv_lens": _lens(n)}
    if "doc_ids" in kw:
        kw["doc_ids"] = (torch.arange(S, device="cuda") >= 128).to(torch.int32).expand(B, S).contiguous()
    q, k, v = _inputs(dt, 4)
    k[:, :, n:] = value
    v[:, :, n:] = value
    seen = visible(B, S, S, **{x: y for x, y in kw.items() if x != "softcap"})[0]
    ref, bound = reference(q, k, v, D ** -0.5, **kw)
    for _ in range(20):
        close(fpkern.score_attention(q, k, v, D ** -0.5, **kw), ref, bound)
    v[:, :, 5, 3] = value
    sees = seen[:, :, 5][:, None].expand(B, H, S)
    clean = torch.ones_like(q, dtype=torch.bool)
    clean[..., 3] = ~sees
    for _ in range(20):
        out = fpkern.score_attention(q, k, v, D ** -0.5, **kw)
        assert not torch.isfinite(out[..., 3][sees]).any()
        assert ((out.double() - ref).abs() <= bound)[clean].all()
    assert fpkern.poll_status() == 0
