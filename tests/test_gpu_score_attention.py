"""GPU: score attention (capped, biased and masked scores, grouped heads, caches) against its
definition in 64 bits, within the bound derived in _score_ref.py."""

import ctypes

import pytest
import torch

from fusionpass_b200 import _lib, fpkern
from tests._score_ref import close, reference, visible

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32

# B, H, Hk, Sq, Sk, D.  Tiles of 128 queries and keys, two query tiles a CTA, two heads a CTA,
# keys shared by several CTAs; sizes around a tile
PROMPTS = [(2, 2, 2, 128, 128, 64), (1, 4, 2, 100, 100, 16), (1, 4, 1, 70, 300, 32), (1, 3, 3, 300, 300, 128),
           (2, 2, 1, 257, 513, 128), (1, 2, 2, 640, 640, 64), (1, 1, 1, 130, 4000, 128), (1, 2, 2, 17, 1001, 64),
           (1, 6, 2, 129, 127, 32)]
# rows of a group in one decoding tile: 1 token, several, 16 rows; one key; keys around a chunk and a tile
TOKENS = [(2, 4, 2, 1, 1, 64), (3, 8, 2, 1, 300, 128), (1, 16, 1, 1, 5000, 128), (2, 4, 4, 5, 130, 32),
          (2, 2, 1, 8, 1000, 16), (1, 1, 1, 16, 17, 64), (2, 3, 3, 1, 129, 128), (5, 2, 2, 2, 15, 64)]

MASKS = ["none", "causal", "cap", "bias", "causal_cap_bias", "window", "causal_window", "prefix", "prefix_lens_window",
         "docs", "docs_mixed", "lens", "all", "negative_scale", "zero_scale"]


def _mask(name, B, H, Sq, Sk, g):
    kw = {}
    rnd = lambda lo, hi, *s: torch.randint(lo, max(hi, lo + 1), s, generator=g, device="cuda").to(torch.int32)  # noqa: E731
    if name in ("causal", "causal_cap_bias", "causal_window", "prefix", "prefix_lens_window", "all"):
        kw["causal"] = True
    if name in ("cap", "causal_cap_bias", "all"):
        kw["softcap"] = 5.0
    if name in ("bias", "causal_cap_bias", "all"):
        kw["slopes"] = torch.rand(H, generator=g, device="cuda") * 0.3
    if name in ("window", "causal_window", "prefix_lens_window"):
        kw["window"] = max(1, Sk // 5)
    if name == "all":
        kw["window"] = max(1, Sk // 2)
    if name in ("prefix", "all"):
        kw["prefix"] = Sk // 3
    if name == "prefix_lens_window":
        kw["prefix"] = rnd(0, Sk + 5, B)
    if name in ("docs", "all"):
        kw["doc_ids"] = rnd(0, 3, B, Sk).sort(1).values
    if name == "docs_mixed":
        kw["doc_ids"] = rnd(-1, 3, B, Sk)
    if name in ("lens", "all"):
        kw["kv_lens"] = rnd(0, Sk + 1, B)
    return kw


def _inputs(B, H, Hk, Sq, Sk, D, dt, g, wide=1.0):
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    return (r(B, H, Sq, D) * wide).to(dt), r(B, Hk, Sk, D).to(dt), r(B, Hk, Sk, D).to(dt)


def _scale(name, D):
    return {"negative_scale": -D ** -0.5, "zero_scale": 0.0}.get(name, D ** -0.5)


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("shape", PROMPTS + TOKENS)
@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_against_definition(dt, shape, mask):
    B, H, Hk, Sq, Sk, D = shape
    g = torch.Generator(device="cuda").manual_seed(sum(shape) * 31 + len(mask))
    q, k, v = _inputs(*shape, dt, g, 3.0 if "cap" in mask else 1.0)
    kw = _mask(mask, B, H, Sq, Sk, g)
    scale = _scale(mask, D)
    ref, bound = reference(q, k, v, scale, **kw)
    out = fpkern.score_attention(q, k, v, scale, **kw)
    assert out.shape == q.shape and out.dtype == dt
    close(out, ref, bound)
    seen = visible(B, Sq, Sk, **{x: y for x, y in kw.items() if x not in ("softcap", "slopes")})[0]
    empty = ~seen.any(-1)[:, None, :, None].expand_as(out)
    assert out[empty].eq(0).all()
    assert fpkern.poll_status() == 0


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("shape", [(2, 2, 2, 200, 300, 64), (1, 4, 2, 100, 260, 128), (2, 8, 2, 1, 300, 128),
                                   (2, 2, 2, 7, 300, 32), (1, 1, 1, 130, 4000, 128)])
@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_what_is_not_seen_may_hold_anything(dt, shape, value):
    """Keys and values behind the lengths, ahead of the queries and in other documents hold
    NaN or infinities: rows that do not see them are as if they were not there, rows that see
    a value that is not finite get it."""
    B, H, Hk, Sq, Sk, D = shape
    g = torch.Generator(device="cuda").manual_seed(7)
    q, k, v = _inputs(*shape, dt, g)
    lens = torch.tensor([Sk - 41, Sk // 2 + 3][:B], device="cuda", dtype=torch.int32)
    ids = (torch.arange(Sk, device="cuda") // 90).to(torch.int32).expand(B, Sk).contiguous()
    for kw in ({"kv_lens": lens}, {"causal": True, "kv_lens": lens}, {"doc_ids": ids}, {"causal": True, "doc_ids": ids}):
        seen = visible(B, Sq, Sk, **kw)[0]
        kk, vv = k.clone(), v.clone()
        never = ~seen.any(1)
        kk.transpose(1, 2)[never] = value
        vv.transpose(1, 2)[never] = value
        ref, bound = reference(q, kk, vv, D ** -0.5, **kw)
        close(fpkern.score_attention(q, kk, vv, D ** -0.5, **kw), ref, bound)
        # a value that some rows see and others do not
        j = Sk // 2 - 20
        vv[:, :, j, 3] = value
        out = fpkern.score_attention(q, kk, vv, D ** -0.5, **kw)
        sees = seen[:, :, j][:, None, :].expand(B, H, Sq)
        assert not torch.isfinite(out[..., 3][sees]).any()
        clean = torch.ones_like(out, dtype=torch.bool)
        clean[..., 3] = ~sees
        assert ((out.double() - ref).abs() <= bound)[clean].all()


@pytest.mark.parametrize("D", [64, 128])
def test_many_partly_seen_tiles_with_infinities(D):
    """More such tiles than the kernel notes key by key."""
    B, H, Sq, Sk = 1, 1, 256, 128 * 40
    g = torch.Generator(device="cuda").manual_seed(9)
    q, k, v = _inputs(B, H, H, Sq, Sk, D, F16, g)
    q, k, v = (t.repeat(1, 160, 1, 1) for t in (q, k, v))  # more blocks than SMs: no split
    ids = torch.zeros(B, Sk, device="cuda", dtype=torch.int32)
    ids[:, ::2] = 1
    v[:, :, ::128, 5] = float("inf")  # even keys: only documents of id 1 see them
    out = fpkern.score_attention(q, k, v, 0.125, doc_ids=ids)
    row = ids[0, Sk - Sq:] == 1
    assert torch.isinf(out[:, :, row, 5]).all() and torch.isfinite(out[:, :, ~row]).all()
    vc = v.clone()
    vc[:, :, ::128, 5] = 0
    ref, bound = reference(q[:, :1], k[:, :1], vc[:, :1], 0.125, doc_ids=ids)
    close(out[:, :1, ~row], ref[:, :, ~row], bound[:, :, ~row])


@pytest.mark.parametrize("D", [64, 128])
def test_many_tiles_seen_whole_by_one_query_tile_and_in_part_by_the_other(D):
    """The infinities of V are cleared for the tile that sees it in part; the other still gets them."""
    B, Sq, Sk = 1, 256, 128 * 40
    g = torch.Generator(device="cuda").manual_seed(10)
    q, k, v = _inputs(B, 1, 1, Sq, Sk, D, F16, g)
    q, k, v = (t.repeat(1, 160, 1, 1) for t in (q, k, v))
    ids = torch.zeros(B, Sk, device="cuda", dtype=torch.int32)
    ids[:, -128::2] = 1  # the second query tile: documents 0 and 1 by turns; all other keys and rows: 0
    v[:, :, :Sk - 256:128, 5] = float("inf")
    out = fpkern.score_attention(q, k, v, 0.125, doc_ids=ids)
    row = ids[0, Sk - Sq:] == 0
    assert torch.isinf(out[:, :, row, 5]).all() and torch.isfinite(out[:, :, ~row]).all()
    assert torch.isfinite(out[..., :5]).all() and torch.isfinite(out[..., 6:]).all()


@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("shape", [(1, 2, 2, 200, 300, 64), (2, 8, 2, 1, 300, 128), (1, 1, 1, 130, 4000, 128)])
def test_scores_of_nan_and_infinity(dt, shape):
    """A query with a NaN gives NaN in its own row alone, at every key column."""
    B, H, Hk, Sq, Sk, D = shape
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = _inputs(*shape, dt, g)
    ref, bound = reference(q, k, v, D ** -0.5)
    qq = q.clone()
    qq[0, 0, 0, 1] = float("nan")
    out = fpkern.score_attention(qq, k, v, D ** -0.5)
    assert torch.isnan(out[0, 0, 0]).all()
    ok = torch.ones(B, H, Sq, dtype=torch.bool, device="cuda")
    ok[0, 0, 0] = False
    assert ((out.double() - ref).abs() <= bound)[ok].all()
    for j in (0, 1, 8, Sk - 1):  # each column of a group of eight pairs
        kk = k.clone()
        kk[:, :, j, 0] = float("nan")
        assert torch.isnan(fpkern.score_attention(q, kk, v, D ** -0.5)).all()


def test_smallest_and_largest_caps():
    for dt, caps in ((F16, (0.01, 1.0, 1000.0)), (BF16, (0.01, 1000.0)), (F32, (0.01, 1000.0, 1e6, 1e30))):
        for shape in ((1, 2, 2, 150, 300, 64), (1, 4, 2, 1, 300, 128)):
            q, k, v = _inputs(*shape, dt, torch.Generator(device="cuda").manual_seed(8), 4.0)
            for cap in caps:
                ref, bound = reference(q, k, v, 0.3, softcap=cap, causal=True)
                if cap > 1000:  # tanh of f32 is within an ulp: no term of the cap itself
                    ref, bound = reference(q, k, v, 0.3, causal=True)  # the cap is a million scores away
                close(fpkern.score_attention(q, k, v, 0.3, softcap=cap, causal=True), ref, bound)


def test_large_and_far_scores():
    """Running maxima that grow and fall by far more than the rescaling threshold."""
    B, H, Sq, Sk, D = 1, 2, 200, 1000, 64
    for dt in (F16, BF16, F32):
        g = torch.Generator(device="cuda").manual_seed(11)
        q, k, v = _inputs(B, H, H, Sq, Sk, D, dt, g, 8.0)
        k = (k * torch.linspace(0.1, 4.0, Sk, device="cuda")[:, None].to(dt)).to(dt)
        for kw in ({}, {"causal": True}, {"softcap": 50.0}, {"slopes": torch.tensor([0.5, 4.0], device="cuda")}):
            for kk in (k, k.flip(2)):
                ref, bound = reference(q, kk, v, 0.5, **kw)
                close(fpkern.score_attention(q, kk, v, 0.5, **kw), ref, bound)


@pytest.mark.parametrize("dt", [F16, F32])
def test_strided_views_and_out(dt):
    B, H, S, D = 2, 4, 150, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn(B, S, 3, H, D, generator=g, device="cuda").to(dt)
    q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
    ref, bound = reference(q, k, v, 0.125, causal=True)
    close(fpkern.score_attention(q, k, v, 0.125, causal=True), ref, bound)
    buf = torch.full((B, S + 2, H, D), 7.0, device="cuda", dtype=dt)  # heads merged, rows behind the last
    out = fpkern.score_attention(q, k, v, 0.125, causal=True, out=buf[:, :S].transpose(1, 2))
    close(out, ref, bound)
    assert buf[:, S:].eq(7).all() and out.data_ptr() == buf.data_ptr()
    # strides and bases that are copied: transposed D, an odd base, an expanded head
    close(fpkern.score_attention(q.transpose(2, 3).contiguous().transpose(2, 3), k, v, 0.125, causal=True), ref, bound)
    odd = torch.randn(B * H * S * D + 1, generator=g, device="cuda").to(dt)[1:].view(B, H, S, D)
    ref2, bound2 = reference(odd, k, v, 0.125)
    close(fpkern.score_attention(odd, k, v, 0.125), ref2, bound2)
    ke, ve = k[:, :1].expand(B, H, S, D), v[:1].expand(B, H, S, D)
    ref3, bound3 = reference(q, ke, ve, 0.125)
    close(fpkern.score_attention(q, ke, ve, 0.125), ref3, bound3)
    one = q[:, :, 7:8]
    ref4, bound4 = reference(one, k, v, 0.125, causal=True)
    close(fpkern.score_attention(one, k, v, 0.125, causal=True), ref4, bound4)


def test_lengths_and_prefixes_out_of_range_are_clamped():
    q, k, v = _inputs(4, 2, 2, 40, 100, 64, F16, torch.Generator(device="cuda").manual_seed(1))
    lens = torch.tensor([-5, 0, 100, 2 ** 31 - 1], device="cuda", dtype=torch.int32)
    pre = torch.tensor([2 ** 31 - 1, 5, -7, 50], device="cuda", dtype=torch.int32)
    for qq in (q, q[:, :, :1]):
        out = fpkern.score_attention(qq, k, v, 0.125, causal=True, kv_lens=lens, prefix=pre)
        ref, bound = reference(qq, k, v, 0.125, causal=True, kv_lens=lens, prefix=pre)
        close(out, ref, bound)
        assert out[:2].eq(0).all()


@pytest.mark.parametrize("B,H,Hk,Sq,Sk,D", [(1, 1, 1, 1, 60, 64), (7, 4, 2, 1, 1500, 64), (128, 4, 4, 1, 300, 32),
                                            (129, 2, 2, 1, 300, 32), (100, 2, 1, 3, 700, 16), (3, 16, 1, 1, 9000, 128)])
def test_decoding_unequal_caches(B, H, Hk, Sq, Sk, D):
    """One line of work over sequences from empty to full; all of it on a few of them; none at all."""
    g = torch.Generator(device="cuda").manual_seed(B + Sk)
    q, k, v = _inputs(B, H, Hk, Sq, Sk, D, BF16, g)
    some = torch.randint(0, Sk + 1, (B,), generator=g, device="cuda").to(torch.int32)
    one = torch.zeros(B, device="cuda", dtype=torch.int32)
    one[B // 2] = Sk
    short = torch.randint(0, 4, (B,), generator=g, device="cuda").to(torch.int32)
    for lens in (some, one, short, torch.zeros_like(one), torch.full_like(one, Sk), some // 2):
        for kw in ({}, {"causal": True, "window": 200}, {"causal": True, "window": 100, "prefix": 130}):
            ref, bound = reference(q, k, v, 0.2, kv_lens=lens, **kw)
            out = torch.full_like(q, 7.0)
            close(fpkern.score_attention(q, k, v, 0.2, kv_lens=lens, out=out, **kw), ref, bound)


def test_no_keys_no_queries():
    for dt in (F16, F32):
        q = torch.randn(2, 4, 5, 64, device="cuda").to(dt)
        k = torch.empty(2, 2, 0, 64, device="cuda", dtype=dt)
        out = torch.full_like(q, 7.0)
        assert fpkern.score_attention(q, k, k, 1.0, out=out).eq(0).all()
        ids = torch.empty(2, 0, device="cuda", dtype=torch.int32)
        assert fpkern.score_attention(q, k, k, 1.0, doc_ids=ids, causal=True).eq(0).all()
        assert fpkern.score_attention(q[:, :, :0], q, q, 1.0).shape == (2, 4, 0, 64)
        assert fpkern.score_attention(q[:0], q[:0], q[:0], 1.0).shape == (0, 4, 5, 64)


def test_streams_and_two_captured_graphs():
    """Calls with workspaces captured into two graphs and replayed on two streams at once."""
    g = torch.Generator(device="cuda").manual_seed(5)
    a = _inputs(1, 2, 2, 130, 4000, 128, F16, g)
    b = _inputs(2, 8, 2, 1, 3000, 128, BF16, g)
    ids = (torch.arange(4000, device="cuda") // 1500).to(torch.int32)[None].contiguous()
    calls = [lambda: fpkern.score_attention(*a, 0.1, causal=True, doc_ids=ids),
             lambda: fpkern.score_attention(*b, 0.1, causal=True, softcap=20.0)]
    want = [reference(*a, 0.1, causal=True, doc_ids=ids), reference(*b, 0.1, causal=True, softcap=20.0)]
    graphs, outs = [], []
    for call in calls:
        call()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(call())
        graphs.append(gr)
    side = torch.cuda.Stream()
    for _ in range(5):
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
            again = calls[0]()
        torch.cuda.current_stream().wait_stream(side)
    for o, (ref, bound) in zip(outs + [again], want + [want[0]]):
        close(o, ref, bound)
    assert torch.equal(again, outs[0])  # the same bits, whatever ran beside it
    assert fpkern.poll_status() == 0


def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 elements: the last sequence, at its far end."""
    B, Hk, Sk, D = 3, 8, 1 << 20, 128  # 3.2e9 elements of k and of v each
    k = torch.zeros(B, Hk, Sk, D, device="cuda", dtype=F16)
    v = torch.zeros(B, Hk, Sk, D, device="cuda", dtype=F16)
    g = torch.Generator(device="cuda").manual_seed(4)
    for t in (k, v):
        t[-1, :, -3000:] = torch.randn(Hk, 3000, D, generator=g, device="cuda").to(F16)
    for Sq in (1, 40):
        q = torch.randn(B, 2 * Hk, Sq, D, generator=g, device="cuda").to(F16)
        out = fpkern.score_attention(q, k, v, 0.1, causal=True, window=2000)
        ref, bound = reference(q[-1:], k[-1:, :, -3000:], v[-1:, :, -3000:], 0.1, causal=True, window=2000)
        close(out[-1:], ref, bound)
        assert out[0].eq(0).all()


def test_refusals():
    q = torch.randn(2, 4, 8, 64, device="cuda").half()
    k = torch.randn(2, 2, 20, 64, device="cuda").half()
    call = lambda *a, **kw: fpkern.score_attention(*a, **kw)  # noqa: E731
    for bad, match in ((lambda: call(q[0], k, k, 1.0), r"\[B, heads, S, D\]"), (lambda: call(q, k, k.float(), 1.0), "dtype"),
                       (lambda: call(q.double(), k.double(), k.double(), 1.0), "dtype"),
                       (lambda: call(q, k, k[:, :, :5], 1.0), "shape"), (lambda: call(q, k[:1], k[:1], 1.0), "batch"),
                       (lambda: call(q[:, :3], k, k, 1.0), "heads"),
                       (lambda: call(q[..., :40], k[..., :40], k[..., :40], 1.0), "head dim"),
                       (lambda: call(q, k, k, float("nan")), "scale"), (lambda: call(q, k, k, 1.0, softcap=0.0), "softcap"),
                       (lambda: call(q, k, k, 1.0, softcap=float("inf")), "softcap"),
                       (lambda: call(q, k, k, 1.0, softcap=1001.0), "f32 only"),
                       (lambda: call(q, k, k, 1.0, window=0), "window"), (lambda: call(q, k, k, 1.0, prefix=-1), "prefix"),
                       (lambda: call(q, k, k, 1.0, slopes=torch.ones(2, device="cuda")), "slopes"),
                       (lambda: call(q, k, k, 1.0, kv_lens=torch.ones(2, device="cuda", dtype=torch.int64)), "kv_lens"),
                       (lambda: call(q, k, k, 1.0, prefix=torch.ones(3, device="cuda", dtype=torch.int32)), "prefix"),
                       (lambda: call(q, k, k, 1.0, doc_ids=torch.ones(2, 8, device="cuda", dtype=torch.int32)), "doc_ids"),
                       (lambda: call(q.clone().requires_grad_(), k, k, 1.0), "gradient"),
                       (lambda: call(q, k, k, 1.0, out=torch.empty(2, 4, 8, 128, device="cuda").half()[..., ::2]), "out")):
        with pytest.raises(ValueError, match=match):
            bad()
    with pytest.raises(RuntimeError, match="CUDA"):
        call(q.cpu(), k, k, 1.0)
    lib = _lib.load()
    d = _lib.ScoreDesc(size=ctypes.sizeof(_lib.ScoreDesc), version=_lib.FPK_ABI_VERSION, dtype=_lib.FPK_F16, head_dim=64,
                       batch=2, heads=4, kv_heads=3, q_len=8, k_len=20, scale=1.0)
    assert lib.fpk_score_attention_workspace(ctypes.byref(d)) == _lib.FPK_ERR_INVALID  # 4 heads over 3
    d.kv_heads = 2
    need = lib.fpk_score_attention_workspace(ctypes.byref(d))
    assert need >= 0
    p = ctypes.c_void_p(q.data_ptr())
    fwd = lambda: lib.fpk_score_attention_fwd(ctypes.byref(d), p, p, p, p, None, 0, None)  # noqa: E731
    assert fwd() == _lib.FPK_ERR_ALIGN  # strides of zero
    for f in (d.q_strides, d.k_strides, d.v_strides, d.o_strides):
        f[0], f[1], f[2] = 8 * 64, 64, 64
    d.q_len, d.k_len = 1, 20000
    if lib.fpk_score_attention_workspace(ctypes.byref(d)) > 0:
        assert fwd() == _lib.FPK_ERR_INVALID  # the workspace is missing
    d.head_dim = 48
    assert fwd() == _lib.FPK_ERR_UNSUPPORTED


@pytest.mark.parametrize("scale, cap", [(3e38, None), (1.0, 1e-39), (1e10, 1e-29)])
def test_factors_beyond_f32_are_refused(scale, cap):
    q = torch.randn(1, 2, 4, 64, device="cuda")
    for t in (q, q.half()):
        with pytest.raises(ValueError, match="softcap" if cap else "scale"):
            fpkern.score_attention(t, t, t, scale, softcap=cap)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sq", [1, 200])
def test_smallest_cap(dt, sq):
    """A cap so small that every score is one of +-cap (or 0): the weights are all but equal."""
    g = torch.Generator(device="cuda").manual_seed(sq)
    q, k, v = (torch.randn(1, 2, n, 64, generator=g, device="cuda").to(dt) for n in (sq, 300, 300))
    k[:, :, 7] = 0  # a score of 0
    o = fpkern.score_attention(q, k, v, 1.0, softcap=1e-37)
    want = v.double().mean(2, keepdim=True).expand(1, 2, sq, 64)
    # the weights are 1 and their sum 300, exactly; sums in f32 (300 2^-24 of the largest |v|), one rounding
    room = 2.0 * torch.finfo(dt).eps / 2 * want.abs() + 300 * 2.0 ** -24 * v.double().abs().max()
    assert ((o.double() - want).abs() <= room).all()


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("kw", [{}, {"causal": True}, {"causal": True, "window": 150, "prefix": 37}, {"softcap": 5.0}],
                         ids=["both_sides", "causal", "window_prefix", "cap"])
@pytest.mark.parametrize("Sq, Sk", [(400, 400), (70, 700), (513, 2000)])
def test_slopes_of_all_sizes(dt, D, kw, Sq, Sk):
    """Slopes of 0, negative, small, large; one of them a value of 24 bits; two heads of a CTA with their own."""
    g = torch.Generator(device="cuda").manual_seed(Sq + D)
    q, k, v = (torch.randn(1, h, n, D, generator=g, device="cuda").to(dt) for h, n in ((6, Sq), (3, Sk), (3, Sk)))
    slopes = torch.tensor([0.0, 1e-6, -0.02, 1 / 3, 5.0, 300.0], device="cuda")
    ref, bound = reference(q, k, v, D ** -0.5, slopes=slopes, **kw)
    close(fpkern.score_attention(q, k, v, D ** -0.5, slopes=slopes, **kw), ref, bound)


@pytest.mark.parametrize("slope", [1e9, 1e27, 1e29, 1e31, 1e36])
@pytest.mark.parametrize("cap", [None, 5.0])
@pytest.mark.parametrize("D", [64, 128])
def test_huge_slopes_leave_the_own_key(slope, cap, D):
    """exp of the distance's bias is 0 for every key but the query's own, whose weight is 1: its value, exactly."""
    g = torch.Generator(device="cuda").manual_seed(D)
    q, k, v = (torch.randn(1, 2, 520, D, generator=g, device="cuda").half() for _ in range(3))
    slopes = torch.tensor([slope, 1.0], device="cuda")
    for causal in (False, True):
        o = fpkern.score_attention(q, k, v, D ** -0.5, softcap=cap, slopes=slopes, causal=causal)
        assert torch.equal(o[:, 0], v[:, 0]) and torch.isfinite(o).all()


def test_slopes_of_nan_stay_in_their_heads():
    g = torch.Generator(device="cuda").manual_seed(1)
    for D, Sq in ((64, 300), (128, 300), (128, 100)):
        q, k, v = (torch.randn(1, h, n, D, generator=g, device="cuda").half() for h, n in ((4, Sq), (2, 300), (2, 300)))
        slopes = torch.tensor([0.1, float("nan"), 0.2, 0.3], device="cuda")
        o = fpkern.score_attention(q, k, v, D ** -0.5, slopes=slopes, causal=True)
        ref, bound = reference(q, k, v, D ** -0.5, slopes=torch.tensor([0.1, 0.1, 0.2, 0.3], device="cuda"), causal=True)
        assert torch.isnan(o[:, 1]).all()
        for h in (0, 2, 3):
            close(o[:, h], ref[:, h], bound[:, h])
