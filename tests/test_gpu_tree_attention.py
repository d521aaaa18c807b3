"""GPU: tree attention against its definition in 64 bits, within the bound derived in _draft_ref.py."""

import pytest
import torch

from fusionpass_b200 import fpkern
from tests._draft_ref import close, quantised, sight, tree_reference

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32

# B, H, Hk, T, N, D: one row, single tokens, rows around the blocks of 16, 32, 64 and 128, trees of one word
# of bits and of all eight, keys around chunks and tiles, trees as large as the cache
SHAPES = [(1, 1, 1, 1, 1, 16), (2, 4, 2, 1, 300, 64), (1, 16, 1, 1, 5000, 128), (3, 8, 2, 8, 257, 128),
          (2, 6, 3, 21, 333, 32), (1, 4, 4, 64, 64, 64), (1, 8, 1, 40, 1000, 16), (2, 4, 1, 100, 129, 128),
          (1, 2, 2, 256, 256, 32), (1, 8, 8, 33, 5000, 64), (1, 64, 8, 16, 4000, 128), (2, 3, 1, 43, 700, 128),
          (3, 2, 2, 17, 130, 16), (2, 16, 2, 65, 1025, 64), (1, 32, 1, 256, 2000, 128),
          # rows 9 to 16, 17 to 32 and 33 of every head dim; more blocks than CTAs, many parts a row
          (2, 10, 1, 1, 300, 16), (2, 12, 1, 1, 300, 32), (1, 4, 1, 4, 700, 64), (2, 13, 1, 1, 900, 128),
          (1, 4, 1, 8, 300, 16), (1, 5, 1, 5, 400, 32), (2, 8, 1, 4, 1300, 64), (1, 2, 1, 15, 260, 128),
          (2, 11, 1, 3, 500, 16), (1, 11, 1, 3, 500, 32), (1, 11, 1, 3, 2500, 128), (40, 20, 20, 2, 140, 32),
          (30, 30, 10, 12, 300, 16), (1, 1, 1, 1, 60000, 64),
          # many sequences: lengths added up beforehand
          (257, 2, 1, 2, 140, 16), (1100, 1, 1, 1, 40, 32)]
TREES = ["tree", "chain", "star", "forest", "ragged", "outside"]


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _parents(kind, B, T, g):
    i = torch.arange(T, device="cuda")
    if kind == "chain":
        p = (i - 1).expand(B, T)
    elif kind == "star":
        p = torch.where(i > 0, 0, -1).expand(B, T)
    else:
        p = (torch.rand(B, T, generator=g, device="cuda") * i).long()
        if kind == "forest":  # values that are no earlier node make a root
            odd = torch.rand(B, T, generator=g, device="cuda") < 0.3
            p = torch.where(odd, i + torch.randint(0, 3, (B, T), generator=g, device="cuda"), p)
            p = torch.where(torch.rand(B, T, generator=g, device="cuda") < 0.1, -2147483648, p)
        else:
            p = torch.where(i > 0, p, -1)
    return p.to(torch.int32).contiguous()


def _inputs(shape, dt, q8, kind, g):
    B, H, Hk, T, N, D = shape
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    q, k, v = (1.5 * r(B, H, T, D)).to(dt), r(B, Hk, N, D), r(B, Hk, N, D)
    kw = {}
    if q8:
        (k, kw["k_scale"]), (v, kw["v_scale"]) = quantised(k), quantised(v * (1.5 * r(B, Hk, N, 1)).exp())
    else:
        k, v = k.to(dt), v.to(dt)
    past = torch.full((B,), N - T, dtype=torch.int32, device="cuda")
    lens = None
    if kind == "ragged":
        past = torch.randint(0, N - T + 1, (B,), generator=g, device="cuda").to(torch.int32)
        lens = torch.randint(0, T + 2, (B,), generator=g, device="cuda").to(torch.int32)
        lens[0] = 0 if B > 2 else T
    if kind == "outside":
        past = i32(-3, N - T + 2, N + 5).repeat(B)[:B]
    return q, k, v, _parents(kind, B, T, g), past, lens, kw


@pytest.mark.parametrize("kind", TREES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_against_definition(dt, q8, shape, kind):
    B, H, Hk, T, N, D = shape
    g = torch.Generator(device="cuda").manual_seed(sum(shape) * 31 + len(kind))
    q, k, v, parents, past, lens, kw = _inputs(shape, dt, q8, kind, g)
    near = sight(parents, past, lens if lens is not None else [T] * B, N)
    ref, bound = tree_reference(q, k, v, D ** -0.5, near, **kw)
    out = fpkern.tree_attention(q, k, v, D ** -0.5, parents, past, tree_lens=lens, **kw)
    assert out.shape == q.shape and out.dtype == dt
    close(out, ref, bound)
    empty = ~near.any(-1)[:, None, :, None].expand(out.shape).cuda()
    assert out[empty].eq(0).all()
    assert fpkern.poll_status() == 0


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
@pytest.mark.parametrize("shape", [(2, 4, 2, 5, 300, 64), (1, 8, 1, 40, 1000, 128)])
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_scales(dt, q8, shape, scale):
    g = torch.Generator(device="cuda").manual_seed(4)
    q, k, v, parents, past, lens, kw = _inputs(shape, dt, q8, "tree", g)
    ref, bound = tree_reference(q, k, v, scale, sight(parents, past, [shape[3]] * shape[0], shape[4]), **kw)
    close(fpkern.tree_attention(q, k, v, scale, parents, past, **kw), ref, bound)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("shape", [(2, 4, 2, 9, 300, 64), (2, 8, 2, 40, 260, 128), (1, 2, 2, 150, 500, 32), (1, 4, 4, 1, 200, 16)])
@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_what_a_node_does_not_see_may_hold_anything(dt, shape, value):
    """Rows behind the tree hold NaN or infinities, and so does one node's value: nodes that do not see it
    are as if it were not there, those that see it get it."""
    B, H, Hk, T, N, D = shape
    g = torch.Generator(device="cuda").manual_seed(7)
    q, k, v, parents, past, lens, _ = _inputs(shape, dt, False, "tree", g)
    past = torch.full_like(past, N - T - 30)
    near = sight(parents, past, [T] * B, N)
    k[:, :, N - 30:] = value
    v[:, :, N - 30:] = value
    ref, bound = tree_reference(q, k, v, D ** -0.5, near)
    close(fpkern.tree_attention(q, k, v, D ** -0.5, parents, past), ref, bound)
    x = T // 2
    v[:, :, N - T - 30 + x, 3] = value
    out = fpkern.tree_attention(q, k, v, D ** -0.5, parents, past)
    sees = near[:, :, N - T - 30 + x].cuda()[:, None].expand(B, H, T)
    assert not torch.isfinite(out[..., 3][sees]).any()
    clean = torch.ones_like(out, dtype=torch.bool)
    clean[..., 3] = ~sees
    assert ((out.double() - ref).abs() <= bound)[clean].all()
    # a key: the whole row of a node that sees it
    k[:, :, N - T - 30 + x, 1] = float("nan")
    out = fpkern.tree_attention(q, k, v, D ** -0.5, parents, past)
    assert torch.isnan(out[sees]).all()
    assert ((out.double() - ref).abs() <= bound)[~sees].all()


@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
@pytest.mark.parametrize("shape", [(2, 4, 2, 9, 300, 64), (2, 8, 2, 40, 260, 128), (1, 2, 2, 150, 500, 32)])
@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_scales_that_are_not_numbers(dt, shape, which):
    """A row written from NaN has the scale NaN: only nodes that see it are NaN."""
    B, H, Hk, T, N, D = shape
    g = torch.Generator(device="cuda").manual_seed(8)
    q, k, v, parents, past, lens, kw = _inputs(shape, dt, True, "tree", g)
    past = torch.full_like(past, N - T - 30)
    near = sight(parents, past, [T] * B, N)
    for s in kw.values():
        s[:, :, N - 30:] = float("nan")
    ref, bound = tree_reference(q, k, v, D ** -0.5, near, **kw)
    close(fpkern.tree_attention(q, k, v, D ** -0.5, parents, past, **kw), ref, bound)
    x = N - T - 30 + T // 2
    kw[which][:, :, x] = float("nan")
    out = fpkern.tree_attention(q, k, v, D ** -0.5, parents, past, **kw)
    sees = near[:, :, x].cuda()[:, None].expand(B, H, T)
    assert torch.isnan(out[sees]).all()
    assert ((out.double() - ref).abs() <= bound)[~sees].all()


@pytest.mark.parametrize("small", [1e-6, 1e-30, 0.0])
@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_values_of_any_magnitude(dt, small):
    """Scales far below and, in part of the keys, far above the others': weights stay in the type's range."""
    shape = (2, 8, 2, 20, 700, 64)
    g = torch.Generator(device="cuda").manual_seed(11)
    q, k, v, parents, past, lens, kw = _inputs(shape, dt, True, "tree", g)
    near = sight(parents, past, [20] * 2, 700)
    kw["v_scale"] *= small
    for _ in range(2):
        ref, bound = tree_reference(q, k, v, 0.125, near, **kw)
        close(fpkern.tree_attention(q, k, v, 0.125, parents, past, **kw), ref, bound)
        kw["v_scale"][:, :, 300] = 2.0


def test_strides_and_shared_parents():
    """Caches laid out [B, N, Hk, D], queries [B, T, H, D], rows off 16 bytes, one tree for all, scales of other
    strides, results in place."""
    B, H, Hk, T, N, D = 3, 8, 2, 12, 200, 64
    g = torch.Generator(device="cuda").manual_seed(5)
    for q8 in (False, True):
        for dt in (F16, F32):
            q, k, v, parents, past, lens, kw = _inputs((B, H, Hk, T, N, D), dt, q8, "ragged", g)
            parents = parents[:1].expand(B, T)
            want = fpkern.tree_attention(q, k, v, 0.125, parents.contiguous(), past, tree_lens=lens, **kw)
            flip = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
            kw2 = {n: flip(t) for n, t in kw.items()}
            for p in (parents, parents[0]):
                assert torch.equal(fpkern.tree_attention(flip(q), flip(k), flip(v), 0.125, p, past, tree_lens=lens, **kw2), want)
            off = torch.zeros(B, Hk, N, D + 3, dtype=k.dtype, device="cuda")
            off[..., 3:] = k
            assert torch.equal(fpkern.tree_attention(q, off[..., 3:], v, 0.125, parents, past, tree_lens=lens, **kw), want)
            out = torch.empty(B, T, H, D, dtype=dt, device="cuda").transpose(1, 2)
            version = out._version
            got = fpkern.tree_attention(q, k, v, 0.125, parents, past, tree_lens=lens, out=out, **kw)
            assert got.data_ptr() == out.data_ptr() and torch.equal(out, want) and out._version > version


def test_one_node_is_score_attention_of_one_token():
    B, H, Hk, N, D = 4, 8, 2, 600, 128
    g = torch.Generator(device="cuda").manual_seed(6)
    q, k, v = (torch.randn(s, generator=g, device="cuda").half() for s in ((B, H, 1, D), (B, Hk, N, D), (B, Hk, N, D)))
    past = i32(0, 17, 599, 300)
    a = fpkern.tree_attention(q, k, v, 0.09, i32(-1), past)
    b = fpkern.score_attention(q, k, v, 0.09, kv_lens=past + 1)
    torch.testing.assert_close(a, b, rtol=2e-3, atol=2e-3)


@pytest.mark.parametrize("T", [1, 20])
def test_a_cache_beyond_32_bits(T):
    """Keys whose offset passes 2^31 elements, 2^32 bytes in f16."""
    N, D = (1 << 20) + 333, 128
    for dt, q8 in ((F16, False), (F16, True)):
        heads = 10 if not q8 else 18
        k, v = (torch.zeros(1, heads, N, D, dtype=torch.int8 if q8 else dt, device="cuda") for _ in range(2))
        g = torch.Generator(device="cuda").manual_seed(3)
        q = torch.randn(1, heads, T, D, generator=g, device="cuda").to(dt)
        last = 400
        new = torch.randint(-127, 128, (2, 1, heads, last, D), generator=g, device="cuda")
        k[:, :, N - last:], v[:, :, N - last:] = ((x if q8 else x / 64).to(k.dtype) for x in new)
        kw = {n: torch.full((1, heads, N), 1 / 64, device="cuda") for n in ("k_scale", "v_scale")} if q8 else {}
        parents = (torch.arange(T, device="cuda") - 1).to(torch.int32)
        out = fpkern.tree_attention(q, k, v, 0.5, parents, i32(N - T), **kw)
        # zero keys have the exponent 0: one of them, N - last times as heavy
        x = q.double() @ k[:, :, N - last:].double().transpose(-1, -2) * (0.5 / (64 if q8 else 1))
        at = torch.arange(last, device="cuda") - (last - T)
        x = x.masked_fill(at > torch.arange(T, device="cuda")[:, None], float("-inf"))
        top = x.amax(-1, keepdim=True).clamp(min=0)
        w = torch.exp(x - top)
        total = w.sum(-1, keepdim=True) + (N - last) * torch.exp(-top)
        ref = (w / total) @ v[:, :, N - last:].double() / (64 if q8 else 1)
        torch.testing.assert_close(out.double(), ref, rtol=4e-3, atol=4e-3)
        del k, v


def test_many_sequences_of_many_lengths():
    """More sequences than one pass of the block that adds lengths up, in both kernels of f16."""
    g = torch.Generator(device="cuda").manual_seed(12)
    for B, T in ((3000, 1), (1500, 40)):
        q, k, v = (torch.randn(B, 1, n, 16, generator=g, device="cuda").half() for n in (T, 300, 300))
        past = torch.randint(0, 300 - T, (B,), generator=g, device="cuda").to(torch.int32)
        chain = (torch.arange(T, device="cuda") - 1).to(torch.int32)
        out = fpkern.tree_attention(q, k, v, 0.25, chain, past)
        seen = torch.arange(300, device="cuda") <= past[:, None, None] + torch.arange(T, device="cuda")[:, None]
        x = (q.double() @ k.double().transpose(-1, -2) * 0.25).masked_fill(~seen[:, None], float("-inf"))
        torch.testing.assert_close(out.double(), torch.softmax(x, -1) @ v.double(), rtol=4e-3, atol=4e-3)


def test_empty_calls():
    q = torch.randn(2, 4, 3, 16, device="cuda").half()
    none = torch.zeros(2, 2, 0, 16, device="cuda").half()
    p, past = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), i32(0, 0)
    assert fpkern.tree_attention(q, none, none, 1.0, p, past).eq(0).all()
    scale = torch.zeros(2, 2, 0, device="cuda")
    assert fpkern.tree_attention(q, none.to(torch.int8), none.to(torch.int8), 1.0, p, past, k_scale=scale, v_scale=scale).eq(0).all()
    assert fpkern.tree_attention(q.float(), none.float(), none.float(), 1.0, p, past).eq(0).all()
    k = torch.randn(2, 2, 5, 16, device="cuda").half()
    wide = torch.randn(2, 4, 90, 16, device="cuda").half()  # on tcgen05
    assert fpkern.tree_attention(wide, none, none, 1.0, torch.zeros(2, 90, dtype=torch.int32, device="cuda"), past).eq(0).all()
    assert fpkern.tree_attention(q[:, :, :0], k, k, 1.0, p[:, :0], past).shape == (2, 4, 0, 16)
    assert fpkern.tree_attention(q, k, k, 1.0, p, past, tree_lens=i32(0, -4)).eq(0).all()


def test_refusals():
    r = lambda *s: torch.randn(*s, device="cuda").half()  # noqa: E731
    q, k, v = r(2, 4, 3, 16), r(2, 2, 9, 16), r(2, 2, 9, 16)
    p, past = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), i32(0, 0)
    k8, s = torch.zeros(2, 2, 9, 16, dtype=torch.int8, device="cuda"), torch.ones(2, 2, 9, device="cuda")
    f = fpkern.tree_attention
    bad = [
        lambda: f(q.double(), k.double(), v.double(), 1.0, p, past),
        lambda: f(q, k.bfloat16(), v.bfloat16(), 1.0, p, past),
        lambda: f(q, k8, k8, 1.0, p, past),
        lambda: f(q, k, v, 1.0, p, past, k_scale=s, v_scale=s),
        lambda: f(q, k8, k8, 1.0, p, past, k_scale=s),
        lambda: f(q, k8, k8, 1.0, p, past, k_scale=s, v_scale=s.half()),
        lambda: f(q, k8, k8, 1.0, p, past, k_scale=s[..., :8], v_scale=s),
        lambda: f(q, k, v[:, :, :8], 1.0, p, past),
        lambda: f(q, k[:1], v[:1], 1.0, p, past),
        lambda: f(q, r(2, 3, 9, 16), r(2, 3, 9, 16), 1.0, p, past),
        lambda: f(r(2, 4, 3, 24), r(2, 2, 9, 24), r(2, 2, 9, 24), 1.0, p, past),
        lambda: f(q[0], k, v, 1.0, p, past),
        lambda: f(q, k, v, float("inf"), p, past),
        lambda: f(q, k, v, float("nan"), p, past),
        lambda: f(q, k, v, 3e38, p, past),
        lambda: f(q, k, v, 1.0, p.long(), past),
        lambda: f(q, k, v, 1.0, p[:, :2], past),
        lambda: f(q, k, v, 1.0, p[:1], past),
        lambda: f(q, k, v, 1.0, p, past.long()),
        lambda: f(q, k, v, 1.0, p, past[:1]),
        lambda: f(q, k, v, 1.0, p, past, tree_lens=past.long()),
        lambda: f(r(2, 4, 257, 16), k, v, 1.0, torch.zeros(2, 257, dtype=torch.int32, device="cuda"), past),
        lambda: f(q, k, v, 1.0, p, past, out=q),
        lambda: f(q, k, v, 1.0, p, past, out=torch.empty(2, 4, 3, 16, device="cuda")),
        lambda: f(q, k, v, 1.0, p, past, out=r(2, 4, 3, 17)[..., 1:]),
        lambda: f(q, k, v, 1.0, p, past, out=r(1, 4, 3, 16).expand(2, 4, 3, 16)),
        lambda: f(q.clone().requires_grad_(), k, v, 1.0, p, past),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    for call in (lambda: f(q.cpu(), k, v, 1.0, p, past), lambda: f(q, k, v, 1.0, p.cpu(), past)):
        with pytest.raises(RuntimeError):
            call()
