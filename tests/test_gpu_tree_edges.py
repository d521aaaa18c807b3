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


def _strict(q, k, v, scale, near, ks=None, vs=None):
    """(out, bound) as tree_reference has them, where the bound of a node knows only the keys that it sees.  What
    f16 holds below 2^-14 in steps of 2^-24 is off by 2^-25 a key at most:
    * of a weight of a 16-bit cache, the largest being 1 or more: 2^-25 |v|;
    * of exp2(y - m) f with 8 bits (y the score and the scale's exponent e, within -60 .. 40, m the largest y, or
      less): 2^-25 * 127 * 2^m, where 2^m is the largest w 2^e.  And y is rounded where the score was: 2^-23 max|e| more."""
    B, H, T, D = q.shape
    Hk, N = k.shape[1:3]
    ref, _ = tree_reference(q, k, v, scale, near, ks, vs)
    near = near.to(q.device)[:, None]
    G = H // Hk
    kd, vd = k.double(), v.double()
    low = torch.zeros(B, Hk, N, device=q.device, dtype=torch.float64)
    if ks is not None:
        kd, vd = kd * ks.double().unsqueeze(-1), vd * vs.double().unsqueeze(-1)
        low = torch.frexp(vs.abs())[1].double().sub(1).clamp(-60, 40)
    kd, vd = (torch.where(near.any(2)[:, :, :, None], t, 0.0).repeat_interleave(G, 1) for t in (kd, vd))
    low = low.repeat_interleave(G, 1).unsqueeze(2)
    qd = q.double()
    x = (qd @ kd.transpose(-1, -2) * scale).masked_fill(~near, float("-inf"))
    terms = torch.where(near, (qd.abs() @ kd.abs().transpose(-1, -2)) * abs(scale), 0.0).amax(-1, keepdim=True)
    big = torch.where(near, x.abs(), 0.0).amax(-1, keepdim=True)
    w = torch.nan_to_num(torch.softmax(x, -1))
    mag = w @ vd.abs()
    u = torch.finfo(q.dtype).eps / 2
    dx = D * 2.0 ** -23 * terms + 4 * 2.0 ** -23 * big
    floor = 0.0
    if q.dtype == F16:
        n = near.sum(-1, keepdim=True)
        if ks is None:
            floor = 2.0 ** -25 * (near.double() @ vd.abs())
        else:
            floor = 2.0 ** -25 * 127 * n * (w * torch.exp2(low)).amax(-1, keepdim=True)
            dx = dx + 2.0 ** -23 * torch.where(near, low.abs(), 0.0).amax(-1, keepdim=True)
    bound = (u + 2.0 ** -23) * ref.abs() + (u + 3 * 2.0 ** -24 + 2 * (4 * 2.0 ** -22 + dx) + N * 2.0 ** -23) * mag + floor
    fi = torch.finfo(q.dtype)
    return ref, bound * (1 + 2 * u) + fi.smallest_normal * fi.eps


def _close(got, ref, bound):
    """Where the result fits its type, and the infinity of its sign where it does not: from 65520 = 2^16 - 2^4 on, half a
    step of 2^5 above the largest number, f16 rounds to infinity."""
    most = torch.finfo(got.dtype).max * (1 + 2.0 ** -12) if got.dtype == F16 else float("inf")
    fits, beyond = ref.abs() + bound < most, ref.abs() - bound >= most
    close(got[fits], ref[fits], bound[fits])
    assert (got[beyond].double() == ref[beyond].sign() * float("inf")).all()


def _tree_call(dt, shape, seed, spread=1.0):
    B, H, Hk, T, N, D = shape
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = (1.5 * _normal(g, B, H, T, D)).to(dt)
    (k, ks), (v, vs) = quantised(_normal(g, B, Hk, N, D)), quantised(_normal(g, B, Hk, N, D) * (spread * _normal(g, B, Hk, N, 1)).exp())
    past = i32(N - T).repeat(B)
    parents = torch.where(torch.arange(T, device="cuda") > 0, 0, -1).to(torch.int32).expand(B, T).contiguous()  # a star
    return q, k, v, ks, vs, parents, past


# mma.sync with up to 8 rows and 16, tcgen05 with 40, 128 and more
LARGE = [(2, 2, 2, 5, 100, 64), (1, 4, 2, 8, 300, 128), (2, 4, 1, 10, 200, 32), (1, 8, 1, 16, 500, 128), (2, 8, 2, 50, 260, 64)]


@pytest.mark.parametrize("large", [65504.0, 1e9, 1e30])
@pytest.mark.parametrize("shape", LARGE)
@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_a_large_value_that_a_node_does_not_see(dt, shape, large):
    """A sibling's value, or one behind the tree, of any finite size: the others' results keep every bit."""
    B, H, Hk, T, N, D = shape
    q, k, v, ks, vs, parents, past = _tree_call(dt, shape, 31)
    past -= 3  # rows behind the tree
    near = sight(parents.cpu(), past.cpu(), [T] * B, N)
    before = fpkern.tree_attention(q, k, v, 0.3, parents, past, k_scale=ks, v_scale=vs)
    ref, bound = _strict(q, k, v, 0.3, near, ks, vs)
    close(before, ref, bound)
    x = T - 2
    vs[:, :, N - 2:] = vs[:, :, N - T - 3 + x] = large / 127
    after = fpkern.tree_attention(q, k, v, 0.3, parents, past, k_scale=ks, v_scale=vs)
    other = torch.arange(T, device="cuda") != x
    assert torch.equal(after[:, :, other], before[:, :, other])
    if dt != F16 or large < 1e30:
        ref, bound = _strict(q, k, v, 0.3, near, ks, vs)
        _close(after, ref, bound)


@pytest.mark.parametrize("shape", LARGE)
@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_values_of_unequal_size(dt, shape):
    """Scales over many powers of two, also where the largest have next to no weight."""
    B, H, Hk, T, N, D = shape
    q, k, v, ks, vs, parents, past = _tree_call(dt, shape, 32, spread=4.0)
    near = sight(parents.cpu(), past.cpu(), [T] * B, N)
    ref, bound = _strict(q, k, v, 0.3, near, ks, vs)
    _close(fpkern.tree_attention(q, k, v, 0.3, parents, past, k_scale=ks, v_scale=vs), ref, bound)
    # one key whose score is far below the others', of a value far above them
    q[..., 0] = 4.0
    k[..., 0] = 0
    k[:, :, 7] = 0
    k[:, :, 7, 0], ks[:, :, 7] = -127, 0.2
    vs.fill_(3 / 127)
    for large in (1e3, 1e6, 1e9, 2.0 ** 46):  # in f16 scales count up to 2^47
        vs[:, :, 7] = large
        ref, bound = _strict(q, k, v, 0.3, near, ks, vs)
        _close(fpkern.tree_attention(q, k, v, 0.3, parents, past, k_scale=ks, v_scale=vs), ref, bound)


def test_values_of_no_size():
    """Rows of zeros (scale 0) that have nearly all of the weight, and caches of nothing else."""
    for dt in (F16, BF16, F32):
        for shape in LARGE:
            B, H, Hk, T, N, D = shape
            q, k, v, ks, vs, parents, past = _tree_call(dt, shape, 33)
            near = sight(parents.cpu(), past.cpu(), [T] * B, N)
            q[..., 0] = 4.0
            k[..., 0] = 0
            k[:, :, :9] = 0
            k[:, :, :9, 0], ks[:, :, :9], vs[:, :, :9] = 127, 0.3, 0.0
            ref, bound = _strict(q, k, v, 0.3, near, ks, vs)
            _close(fpkern.tree_attention(q, k, v, 0.3, parents, past, k_scale=ks, v_scale=vs), ref, bound)
            vs.zero_()
            assert fpkern.tree_attention(q, k, v, 0.3, parents, past, k_scale=ks, v_scale=vs).eq(0).all()


@pytest.mark.parametrize("at", ["early", "near", "tree"])
@pytest.mark.parametrize("heads, T, D", [(1, 1, 64), (2, 6, 16), (4, 12, 128), (1, 60, 64), (8, 40, 32), (16, 4, 128)])
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_values_that_are_not_finite_stay_so_however_the_work_is_cut(dt, q8, heads, T, D, at):
    """A value, or scale, that is infinite or NaN, of a key whose weight vanishes (score -300 against about 0): the elements
    of nodes that see it are not finite, in one sequence (many parts) as among many (few), and no others."""
    N = 3000
    g = torch.Generator(device="cuda").manual_seed(41)
    q, k, v = _normal(g, 1, heads, T, D).to(dt), _normal(g, 1, 1, N, D), _normal(g, 1, 1, N, D)
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    past = N - T - 2
    x = {"early": 100, "near": past - 1, "tree": past}[at]
    k[:, :, x] = 0.0
    k[:, :, x, 0] = -300.0
    kw = {}
    if q8:
        (k, kw["k_scale"]), (v, kw["v_scale"]) = quantised(k), quantised(v)
    else:
        k, v = k.to(dt), v.to(dt)
    parents = (torch.arange(T, device="cuda") - 1).to(torch.int32)  # a chain: every node sees key x
    for value in (float("inf"), -float("inf"), NAN):
        if q8:
            kw["v_scale"][:, :, x] = value
        else:
            v[:, :, x, 5] = value
        for B in (1, 7, 200):
            many = {n: t.expand(B, -1, -1).contiguous() for n, t in kw.items()}
            out = fpkern.tree_attention(q.expand(B, -1, -1, -1).contiguous(), k.expand(B, -1, -1, -1).contiguous(),
                                        v.expand(B, -1, -1, -1).contiguous(), 0.125, parents, i32(past).repeat(B), **many)
            odd = ~torch.isfinite(out)
            if q8:
                assert odd.all()
            else:
                assert odd[..., 5].all() and odd.sum() == odd[..., 5].numel()


@pytest.mark.parametrize("shape", LARGE + [(1, 8, 8, 33, 5000, 64), (1, 32, 1, 100, 2000, 128), (300, 2, 1, 20, 140, 16)])
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_a_workspace_of_any_contents(dt, q8, shape):
    """The allocator's memory holds NaN, infinities or what an earlier call left there: every bit stays."""
    B, H, Hk, T, N, D = shape
    q, k, v, ks, vs, parents, past = _tree_call(dt, shape, 51)
    past[B // 2:] = -T  # and sequences without a key
    kw = dict(k_scale=ks, v_scale=vs) if q8 else {}
    if not q8:
        k, v = ((t.float() * s.unsqueeze(-1)).to(dt) for t, s in ((k, ks), (v, vs)))
    want = fpkern.tree_attention(q, k, v, 0.2, parents, past, **kw)
    torch.cuda.synchronize()
    for fill in (NAN, float("inf"), -float("inf")):
        torch.cuda.empty_cache()
        dirty = [torch.full((n,), fill, device="cuda") for n in (100, 10000, 100000, 1 << 20, 1 << 23, 1 << 25)]
        del dirty
        assert torch.equal(fpkern.tree_attention(q, k, v, 0.2, parents, past, **kw), want)
