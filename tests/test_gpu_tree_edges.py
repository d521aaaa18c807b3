"""GPU: tree attention where one sequence, node or part of the keys must not reach another's result."""

import pytest
import torch

from fusionpass_b200 import fpkern
from tests._draft_ref import close, quantised, sight, tree_reference

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
NAN = float("nan")


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


@pytest.mark.parametrize("heads, nodes", [(1, 12), (1, 40), (4, 40)])
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_rows_behind_the_cache_beside_values_that_are_not_finite(dt, q8, heads, nodes):
    """Sequences in turn: one whose node 15 (or 5) has a value that is no number, one whose tree ends behind the
    cache, so that its node of that number has no row.  Where it would be, memory holds NaN.  Many sequences a CTA."""
    B, D, room, real = 600, 64, 256, 200
    x = 15 if nodes > 15 else 5
    g = torch.Generator(device="cuda").manual_seed(21 + heads + nodes)
    q, k, v = _normal(g, B, heads, nodes, D).to(dt), _normal(g, B, 1, room, D), _normal(g, B, 1, room, D)
    kw = {}
    if q8:
        (k, kw["k_scale"]), (v, kw["v_scale"]) = quantised(k), quantised(v)
        kw["k_scale"][:, :, real:] = kw["v_scale"][:, :, real:] = NAN
        kw["v_scale"][::2, :, 100 + x] = NAN
    else:
        k, v = k.to(dt), v.to(dt)
        k[:, :, real:] = v[:, :, real:] = NAN
        v[::2, :, 100 + x] = NAN
    k, v, kw = k[:, :, :real], v[:, :, :real], {n: s[:, :, :real] for n, s in kw.items()}
    past = i32(100, real - x + 2).repeat(B // 2)
    parents = (torch.arange(nodes, device="cuda") - 1).to(torch.int32)  # a chain: later nodes see the node
    out = fpkern.tree_attention(q, k, v, 0.125, parents, past, **kw)
    assert fpkern.poll_status() == 0
    near = sight(parents[None].expand(2, nodes).cpu(), past[:2].cpu(), [nodes] * 2, real).repeat(B // 2, 1, 1)
    sees = near[:, :, 100 + x].cuda().clone()
    sees[1::2] = False
    finite = torch.where(torch.isfinite(v), v, 0) if not q8 else v
    if q8:
        kw["v_scale"] = torch.where(torch.isfinite(kw["v_scale"]), kw["v_scale"], 0)
    ref, bound = tree_reference(q, k, finite, 0.125, near, **kw)
    sees = sees[:, None].expand(B, heads, nodes)
    assert torch.isnan(out[sees]).all()
    close(out[~sees], ref[~sees], bound[~sees])


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_runs_of_blocks_of_one_key_tile(dt, q8):
    """33 to 128 rows: two warpgroups take every other key tile, so that blocks of one leave the second without
    any.  Long runs of them, with blocks of two and three between, over and over."""
    B, H, T, room, D = 4000, 2, 20, 384, 16
    g = torch.Generator(device="cuda").manual_seed(22)
    q, k, v = _normal(g, B, H, T, D).to(dt), _normal(g, B, 1, room, D), _normal(g, B, 1, room, D)
    kw = {}
    if q8:
        (k, kw["k_scale"]), (v, kw["v_scale"]) = quantised(k), quantised(v)
    else:
        k, v = k.to(dt), v.to(dt)
    past = torch.randint(0, 100, (B,), generator=g, device="cuda")
    past[::37] = 200
    past[5::101] = 350
    past = past.to(torch.int32)
    parents = (torch.arange(T, device="cuda") - 1).to(torch.int32)
    out = fpkern.tree_attention(q, k, v, 0.25, parents, past, **kw)
    near = torch.arange(room, device="cuda") <= past[:, None, None] + torch.arange(T, device="cuda")[:, None]
    ref, bound = tree_reference(q, k, v, 0.25, near, **kw)
    close(out, ref, bound)
    for _ in range(20):
        assert torch.equal(fpkern.tree_attention(q, k, v, 0.25, parents, past, **kw), out)
    assert fpkern.poll_status() == 0
