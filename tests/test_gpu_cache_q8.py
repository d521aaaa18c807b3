"""GPU: the 8-bit cache against its definition: written bits, rows left alone, what is read back,
the rows of an accepted branch."""

import pytest
import torch

from fusionpass_b200 import fpkern
from tests._draft_ref import quantised

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _caches(B, Hk, N, D, g, order="bhnd"):
    """Caches with something in every row; other orders are views of [B, N, Hk, D] or of keys beside values."""
    def q():
        return torch.randint(-127, 128, (B, Hk, N, D), generator=g, device="cuda").to(torch.int8)

    def s():
        return torch.rand(B, Hk, N, generator=g, device="cuda") + 0.5

    if order == "bhnd":
        return q(), q(), s(), s()
    if order == "bnhd":
        return tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q(), q(), s(), s()))
    kv, sc = torch.stack([q(), q()], 3), torch.stack([s(), s()], 3)  # [B, Hk, N, 2, D]
    return kv[..., 0, :], kv[..., 1, :], sc[..., 0], sc[..., 1]


def _written(caches, k, v, past, lens):
    """The caches after the write, by the definition."""
    kc, vc, ks, vs = (t.clone() for t in caches)
    N = kc.shape[2]
    for x, c, s in ((k, kc, ks), (v, vc, vs)):
        q, one = quantised(x)
        for b in range(x.shape[0]):
            for i in range(min(max(int(lens[b]), 0), x.shape[2])):
                to = int(past[b]) + i
                if 0 <= to < N:
                    c[b, :, to], s[b, :, to] = q[b, :, i], one[b, :, i]
    return kc, vc, ks, vs


def same(got, want):
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b, rtol=0.0, atol=0.0, equal_nan=True)


@pytest.mark.parametrize("order", ["bhnd", "bnhd", "pair"])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 16), (2, 3, 9, 5, 32), (3, 2, 40, 40, 64), (2, 2, 300, 77, 128),
                                   (1, 5, 130, 129, 16), (4, 1, 64, 3, 128)])
@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_write(dt, shape, order):
    B, Hk, N, S, D = shape
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    caches = _caches(B, Hk, N, D, g, order)
    k, v = ((torch.randn(B, Hk, S, D, generator=g, device="cuda") * 3).to(dt) for _ in range(2))
    past = torch.randint(0, N - S + 1, (B,), generator=g, device="cuda").to(torch.int32)
    lens = torch.randint(0, S + 1, (B,), generator=g, device="cuda").to(torch.int32)
    for new in (None, lens):
        want = _written(caches, k, v, past, lens if new is not None else [S] * B)
        versions = [t._version for t in caches]
        assert fpkern.cache_write_q8(k, v, *caches, past, new_lens=new) is None
        same(caches, want)
        assert all(t._version > n for t, n in zip(caches, versions))
    # rows of other strides and off 16 bytes are copied first
    wide = torch.zeros(B, S, Hk, D + 1, dtype=dt, device="cuda")
    wide[..., 1:] = k.transpose(1, 2)
    want = _written(caches, k, k, past, [S] * B)
    fpkern.cache_write_q8(wide[..., 1:].transpose(1, 2), wide[..., 1:].transpose(1, 2), *caches, past)
    same(caches, want)


def test_write_leaves_rows_outside_out():
    g = torch.Generator(device="cuda").manual_seed(3)
    caches = _caches(6, 2, 20, 32, g)
    k, v = (torch.randn(6, 2, 7, 32, generator=g, device="cuda") for _ in range(2))
    past = i32(-3, 15, 20, 2147483647, -2147483648, 13)
    lens = i32(7, 100, 3, 7, 7, -1)
    want = _written(caches, k, v, past, lens)
    fpkern.cache_write_q8(k, v, *caches, past, new_lens=lens)
    same(caches, want)


@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_write_of_rows_that_are_not_ordinary(dt):
    """Infinities, NaN, zeros, the smallest and the largest numbers, a row of one value."""
    fi = torch.finfo(dt)
    rows = torch.zeros(9, 16, dtype=dt, device="cuda")
    rows[0, 3] = float("inf")
    rows[1, 5] = float("nan")
    rows[2, 0], rows[2, 1] = float("-inf"), 1.0
    rows[4] = fi.tiny
    rows[5] = fi.max
    rows[6] = -fi.max
    rows[7, 2] = fi.smallest_normal * fi.eps
    rows[8] = torch.linspace(-1, 1, 16).to(dt)
    k = rows.reshape(1, 1, 9, 16)
    caches = _caches(1, 1, 9, 16, torch.Generator(device="cuda").manual_seed(1))
    fpkern.cache_write_q8(k, k, *caches, i32(0))
    want = quantised(k)
    same(caches, (want[0], want[0], want[1], want[1]))
    assert torch.isnan(caches[2][0, 0, :3]).all() and caches[0][0, 0, :3].eq(0).all()


def test_values_in_the_middle_and_next_to_it():
    """127 x / top in the middle of two whole numbers goes to the even one, its neighbours to the nearer."""
    g = torch.Generator(device="cuda").manual_seed(5)
    n = torch.randint(-127, 127, (200, 1), generator=g, device="cuda").float()
    for top in (127.0, 254.0, 1.0, 3.0, 0.7, 1e-30, 1e30):
        mid = ((n.double() + 0.5) * top / 127.0).float()
        up, down = torch.nextafter(mid, mid + top), torch.nextafter(mid, mid - top)
        rows = torch.cat([torch.full_like(mid, top), mid, up, down, -mid, mid * 0.5], 1).repeat(1, 3)[:, :16]
        k = rows.reshape(1, 1, 200, 16).contiguous()
        caches = _caches(1, 1, 200, 16, g)
        fpkern.cache_write_q8(k, k, *caches, i32(0))
        same(caches[:1], quantised(k)[:1])
    for dt in (F16, BF16):  # few digits: many of them lie in the middle
        k = torch.randint(-2000, 2001, (1, 8, 500, 32), generator=g, device="cuda").to(dt)
        k[..., 0] = 127 * 16
        caches = _caches(1, 8, 500, 32, g)
        fpkern.cache_write_q8(k, k, *caches, i32(0))
        same(caches[:1], quantised(k)[:1])


@pytest.mark.parametrize("order", ["bhnd", "bnhd", "pair"])
@pytest.mark.parametrize("shape", [(1, 1, 1, 16), (2, 3, 9, 32), (3, 2, 40, 64), (2, 2, 300, 128), (1, 5, 131, 16)])
@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_read(dt, shape, order):
    B, Hk, N, D = shape
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    kc, vc, ks, vs = _caches(B, Hk, N, D, g, order)
    lens = torch.randint(-1, N + 3, (B,), generator=g, device="cuda").to(torch.int32)
    behind = torch.arange(N, device="cuda") >= lens[:, None]
    ks.transpose(1, 2)[behind] = float("nan")  # what is not read may hold anything
    k, v = fpkern.cache_read_q8(kc, vc, ks, vs, dtype=dt, kv_lens=lens)
    held = ~behind[:, None, :, None]
    same((k, v), (torch.where(held, kc.float() * ks.unsqueeze(-1), 0.0).to(dt),
                  torch.where(held, vc.float() * vs.unsqueeze(-1), 0.0).to(dt)))
    k, v = fpkern.cache_read_q8(kc, vc, ks, vs, dtype=dt)
    same((k, v), ((kc.float() * ks.unsqueeze(-1)).to(dt), (vc.float() * vs.unsqueeze(-1)).to(dt)))
    assert k.is_contiguous() and k.dtype == dt


def _kept(caches, path, counts, past):
    out = []
    for c in caches:
        new = c.clone()
        for b in range(c.shape[0]):
            for i in range(min(max(int(counts[b]), 0), path.shape[1])):
                a, z = int(past[b]) + int(path[b, i]), int(past[b]) + i
                if int(path[b, i]) >= 0 and 0 <= a < c.shape[2] and 0 <= z < c.shape[2]:
                    new[b, :, z] = c[b, :, a]
        out.append(new)
    return out


@pytest.mark.parametrize("order", ["bhnd", "bnhd", "pair"])
@pytest.mark.parametrize("kind", ["branch", "any"])
@pytest.mark.parametrize("shape", [(1, 1, 2, 1, 16), (3, 2, 40, 11, 64), (2, 3, 600, 256, 128), (5, 8, 90, 33, 32)])
def test_keep(shape, kind, order):
    B, Hk, N, P, D = shape
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    caches = list(_caches(B, Hk, N, D, g, order))
    # other types and widths in the same launch: rows of 2, 6 and 512 bytes, another number of heads
    caches += [torch.randn(B, Hk + 1, N, generator=g, device="cuda").half(),
               torch.randn(B, 1, N, 3, generator=g, device="cuda").bfloat16(),
               torch.randn(B, Hk, N, 128, generator=g, device="cuda"),
               torch.randint(0, 2, (B, 2, N, 5), generator=g, device="cuda").bool()]
    past = torch.randint(0, N - P + 1, (B,), generator=g, device="cuda").to(torch.int32)
    counts = torch.randint(0, P + 1, (B,), generator=g, device="cuda").to(torch.int32)
    if kind == "branch":
        path = torch.stack([torch.randperm(P, generator=g, device="cuda") for _ in range(B)])
        path = torch.where(torch.arange(P, device="cuda") < counts[:, None], path, P).sort(1).values
        path = torch.where(path < P, path, -1).to(torch.int32)
    else:  # the same row twice, backwards, outside of the cache
        path = torch.randint(-2, P + N, (B, P), generator=g, device="cuda").to(torch.int32)
        path[:, : P // 2] = torch.randint(0, P, (B, P // 2), generator=g, device="cuda").to(torch.int32)
        counts += 1
        past[0] = -1
    want = _kept(caches, path, counts, past)
    versions = [t._version for t in caches]
    assert fpkern.cache_keep(caches, path, counts, past) is None
    same(caches, want)
    assert all(t._version > n for t, n in zip(caches, versions))


def test_a_cache_beyond_32_bits():
    """Rows whose offset in bytes passes 2^32 (f32 of 4.3 GB) and 2^31 elements of an 8-bit cache."""
    N, D = (1 << 23) + 700, 128
    kc, vc = (torch.zeros(1, 2, N, D, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(1, 2, N, device="cuda") for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(2)
    k, v = (torch.randn(1, 2, 33, D, generator=g, device="cuda") for _ in range(2))
    past = i32(N - 40)
    fpkern.cache_write_q8(k, v, kc, vc, ks, vs, past)
    for x, c, s in ((k, kc, ks), (v, vc, vs)):
        q, one = quantised(x)
        same((c[:, :, N - 40:N - 7], s[:, :, N - 40:N - 7]), (q, one))
    path, counts = torch.arange(0, 33, 4, device="cuda", dtype=torch.int32)[None], i32(9)
    want = _kept([kc[:, :, N - 40:], ks[:, :, N - 40:]], path, counts, i32(0))
    fpkern.cache_keep([kc, ks], path, counts, past)
    same((kc[:, :, N - 40:], ks[:, :, N - 40:]), want)
    assert not kc[:, :, :N - 40].any()
    view = [t[:, 1:, N - 64:] for t in (kc, vc, ks, vs)]
    r, _ = fpkern.cache_read_q8(*view, dtype=F32)
    same((r,), (view[0].float() * view[2].unsqueeze(-1),))


def test_empty_calls():
    g = torch.Generator(device="cuda").manual_seed(1)
    caches = _caches(2, 2, 8, 16, g)
    want = [t.clone() for t in caches]
    none = torch.zeros(2, 2, 0, 16, device="cuda")
    fpkern.cache_write_q8(none, none, *caches, i32(0, 0))
    fpkern.cache_keep(caches, torch.zeros(2, 0, dtype=torch.int32, device="cuda"), i32(1, 1), i32(0, 0))
    fpkern.cache_keep(caches, i32(3, 3)[:, None], i32(0, -1), i32(0, 0))
    same(caches, want)
    empty = tuple(t[:, :, :0] for t in caches)
    k, v = fpkern.cache_read_q8(*empty)
    assert k.shape == v.shape == (2, 2, 0, 16) and k.dtype == F16
    x = torch.randn(2, 2, 3, 16, device="cuda")
    fpkern.cache_write_q8(x, x, *empty, i32(0, 0))


def test_refusals():
    g = torch.Generator(device="cuda").manual_seed(1)
    kc, vc, ks, vs = _caches(2, 2, 8, 16, g)
    k = torch.randn(2, 2, 3, 16, device="cuda")
    past, path, one = i32(0, 0), torch.zeros(2, 3, dtype=torch.int32, device="cuda"), i32(1, 1)
    write = lambda *a, **kw: fpkern.cache_write_q8(*a, **kw)  # noqa: E731
    bad = [
        lambda: write(k.double(), k.double(), kc, vc, ks, vs, past),
        lambda: write(k, k.half(), kc, vc, ks, vs, past),
        lambda: write(k[:, :1], k[:, :1], kc, vc, ks, vs, past),
        lambda: write(k[..., :8], k[..., :8], kc, vc, ks, vs, past),
        lambda: write(k, k, kc.short(), vc, ks, vs, past),
        lambda: write(k, k, kc, vc, ks.half(), vs, past),
        lambda: write(k, k, kc, vc, ks[..., :-1], vs, past),
        lambda: write(k, k, kc, vc[:, :, :4], ks, vs[:, :, :4], past),
        lambda: write(k, k, kc, vc, ks, vs, past.long()),
        lambda: write(k, k, kc, vc, ks, vs, past[:1]),
        lambda: write(k, k, kc, vc, ks, vs, past, new_lens=past.float()),
        lambda: write(k, k, kc, kc, ks, vs, past),
        lambda: write(k, k, kc, vc, ks, ks, past),
        lambda: write(k, k, kc[:1].expand(2, 2, 8, 16), vc, ks, vs, past),
        lambda: write(k, k, torch.zeros(2, 2, 8, 17, dtype=torch.int8, device="cuda")[..., 1:], vc, ks, vs, past),
        lambda: write(k, k, kc.transpose(2, 3).contiguous().transpose(2, 3), vc, ks, vs, past),
        lambda: write(k.clone().requires_grad_(), k, kc, vc, ks, vs, past),
        lambda: fpkern.cache_read_q8(kc, vc, ks, vs, dtype=torch.float64),
        lambda: fpkern.cache_read_q8(kc, vc, ks, vs, dtype="f16"),
        lambda: fpkern.cache_read_q8(kc, vc, ks, vs, kv_lens=past.long()),
        lambda: fpkern.cache_read_q8(kc[..., :8], vc[..., :8], ks, vs),
        lambda: fpkern.cache_keep([], path, one, past),
        lambda: fpkern.cache_keep([ks] * 65, path, one, past),
        lambda: fpkern.cache_keep([kc, kc], path, one, past),
        lambda: fpkern.cache_keep([kc], path.long(), one, past),
        lambda: fpkern.cache_keep([kc], path[0], one, past),
        lambda: fpkern.cache_keep([kc], path, one.long(), past),
        lambda: fpkern.cache_keep([kc], path, one, past[:1]),
        lambda: fpkern.cache_keep([kc], torch.zeros(2, 257, dtype=torch.int32, device="cuda"), one, past),
        lambda: fpkern.cache_keep([kc, ks[:1]], path, one, past),
        lambda: fpkern.cache_keep([kc.transpose(2, 3)], path, one, past),
        lambda: fpkern.cache_keep([ks[:, :1].expand(2, 2, 8)], path, one, past),
    ]
    want = [t.clone() for t in (kc, vc, ks, vs)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(RuntimeError):
        write(k.cpu(), k.cpu(), kc, vc, ks, vs, past)
    same((kc, vc, ks, vs), want)
