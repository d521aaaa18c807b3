"""GPU: RMS norm of a sum of addends and its 8-bit form against the formulas in 64 bits.

Tolerances.  u = eps/2 of the output type (the one rounding at the store, relative to the
value).  In f32 before it, for a row of n columns and k addends: k - 1 roundings of the
sum (relative to the partial sums: the addends are of one sign and size class in each
test's bound, so (k - 1) * 2^-24 * sum|a_i|), n + 3 for the mean square (halved by the square root),
and 4 for the factors.  With n <= 20000 and sums of squares added in several partial sums
of at most n / 32 + 10 terms: below 2^-24 * (n / 64 + 12) relative.
8 bits: the scale carries the same relative error; q may differ by one step from the
rounding in 64 bits (where the value lies near a half), so a value is off by at most half
a step and what the f32 error moves it, (0.5 + 127 * 2^-24 * (n / 64 + 12)) * scale."""

import ctypes

import pytest
import torch

from fusionpass_b200 import _lib, fpkern

pytestmark = pytest.mark.gpu

EPS = 1e-6


def _ref(addends, w, norm=True, eps=EPS):
    s = addends[0].double()
    for t in addends[1:]:
        s = s + t.double()
    r = (s.square().mean(-1, keepdim=True) + eps).rsqrt() if norm else 1.0
    y = s * r
    return (y * w.double() if w is not None else y), s


def _slack(n):
    return 2.0 ** -24 * (n / 64 + 12)


def _inputs(shape, dt, kinds, seed, weight=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    adds = [torch.randn(shape if k == "full" else shape[-1:], generator=g, device="cuda").to(dt) for k in kinds]
    w = (1 + 0.2 * torch.randn(shape[-1], generator=g, device="cuda")).to(dt) if weight else None
    return adds, w


def _mag(adds):
    m = adds[0].double().abs()
    for t in adds[1:]:
        m = m + t.double().abs()
    return m


def _check_y(y, ref, adds, w, n):
    # |y - ref| <= u |ref| + slack |ref| + error of the sum through the factors
    s = _mag(adds)
    sum_err = (len(adds) - 1) * 2.0 ** -24 * s
    rel = torch.finfo(y.dtype).eps / 2 * (1 + 1e-3) + _slack(n)
    r = (ref.abs() + 1e-300) / (adds_sum(adds).abs() + 1e-300)  # the factor r * w of each element
    tiny = torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps
    assert ((y.double() - ref).abs() <= rel * ref.abs() + 2 * sum_err * r + tiny).all()


def adds_sum(adds):
    s = adds[0].double()
    for t in adds[1:]:
        s = s + t.double()
    return s


# one column, one vector, warp rows, block rows of 1, 2 and 4 vectors a thread, rows read twice;
# widths that no vector divides; several leading dims
SHAPES = [(1, 1), (3, 8), (5, 7), (33, 64), (2, 3, 200), (9, 256), (4, 520), (7, 1000), (3, 2049), (16, 4096),
          (2, 8191), (2, 16384), (3, 20001), (2, 40000),
          # more rows than SMs: a resident grid; 32 to 512 threads a row; rows that do not begin on 16 bytes
          (149, 1), (1000, 7), (700, 64), (301, 250), (260, 512), (170, 1000), (163, 1536), (150, 2049), (333, 3001),
          (150, 4096), (149, 6000), (150, 8191), (152, 16376), (149, 16385)]


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_rms_norm_and_sum(shape, dt):
    n = shape[-1]
    for kinds, weight in ((("full",), True), (("full", "full"), True), (("full", "col", "full", "full"), False)):
        adds, w = _inputs(shape, dt, kinds, n + len(kinds), weight)
        y, total = fpkern.add_rms_norm(adds, w, EPS, shape=shape, return_sum=True)
        ref, s = _ref(adds, w)
        assert y.shape == total.shape == torch.Size(shape) and y.dtype == total.dtype == dt
        _check_y(y, ref, adds, w, n)
        u = torch.finfo(dt).eps / 2 * (1 + 1e-3)
        tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
        assert ((total.double() - s).abs() <= u * s.abs() + 3 * 2.0 ** -24 * _mag(adds) * (1 + u) + tiny).all()
    assert torch.equal(fpkern.rms_norm(adds[0], None, EPS), fpkern.add_rms_norm([adds[0]], None, EPS))
    assert fpkern.poll_status() == 0


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_rms_norm_q8(shape, dt):
    n = shape[-1]
    adds, w = _inputs(shape, dt, ("full", "full"), n, True)
    q, scale, total = fpkern.rms_norm_q8(adds, w, EPS, return_sum=True)
    ref, s = _ref(adds, w)
    assert q.dtype == torch.int8 and q.shape == torch.Size(shape) and q.stride(-1) == 1
    assert scale.dtype == torch.float32 and scale.shape == torch.Size(shape[:-1])
    if len(shape) > 1 and shape[-2] > 1:
        assert q.stride(-2) % 16 == 0
    _check_q(q, scale, ref, adds, n)
    assert torch.equal(total, fpkern.add_rms_norm(adds, w, EPS, return_sum=True)[1])
    assert q.abs().amax(-1).eq(127).all()  # the largest magnitude is the 127th step itself


def _check_q(q, scale, ref, adds, n):
    want = ref.abs().amax(-1) / 127
    # the largest element's sum has lost at most (k - 1) 2^-24 of its addends' magnitudes
    lost = (len(adds) - 1) * 2.0 ** -24 * (_mag(adds) / (adds_sum(adds).abs() + 1e-300)).gather(
        -1, ref.abs().argmax(-1, keepdim=True)).squeeze(-1)
    assert ((scale.double() - want).abs() <= (_slack(n) + 2 * lost) * want + 1e-44).all()
    step = want.unsqueeze(-1)
    off = (q.double() * scale.double().unsqueeze(-1) - ref).abs()
    room = (0.5 + 127 * (_slack(n) + 2 * lost.unsqueeze(-1))) * step + 2 * (len(adds) - 1) * 2.0 ** -24 * _mag(adds) * (
        (ref.abs() + 1e-300) / (adds_sum(adds).abs() + 1e-300))
    assert (off <= room + 1e-44).all()


@pytest.mark.parametrize("shape", [(1, 5), (8, 64), (3, 1030), (1001, 1024), (2, 2, 4096), (2, 40000)])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
def test_quantize_q8(shape, dt):
    (x,), _ = _inputs(shape, dt, ("full",), shape[-1], False)
    q, scale = fpkern.quantize_q8(x)
    _check_q(q, scale, x.double(), [x], 1)


@pytest.mark.parametrize("n", [64, 2049, 4096, 40000])
def test_rows_of_zeros_infinities_and_nan(n):
    x = torch.randn(6, n, device="cuda")
    x[0] = 0.0
    x[1, n // 2] = float("inf")
    x[2, n - 1] = float("nan")
    x[3] *= 1e-38  # largest magnitude below 127 of the smallest normal: counts as zero
    x[5, 0] = -float("inf")
    q, scale = fpkern.quantize_q8(x)
    assert scale[0] == 0 and q[0].eq(0).all() and scale[3] == 0 and q[3].eq(0).all()
    for r in (1, 2, 5):
        assert torch.isnan(scale[r]) and q[r].eq(0).all()
    _check_q(q[4:5], scale[4:5], x[4:5].double(), [x[4:5]], 1)
    q, scale = fpkern.rms_norm_q8([x], None, EPS)
    assert scale[0] == 0 and torch.isnan(scale[[1, 2, 5]]).all() and torch.isfinite(scale[4])
    y = fpkern.rms_norm(x, None, EPS)
    assert y[0].eq(0).all() and torch.isnan(y[2]).all()


def test_strided_inputs_streams_and_out():
    big = torch.randn(40, 2, 512, device="cuda").half()
    x, r = big[:, 0], big[::2, 1].repeat_interleave(2, 0)
    w = torch.randn(1024, device="cuda").half()[::2]
    ref, _ = _ref([x, r], w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = torch.empty(40, 512, device="cuda", dtype=torch.float16)
        y = fpkern.add_rms_norm([x, r], w, EPS, out=out)
    torch.cuda.current_stream().wait_stream(side)
    assert y.data_ptr() == out.data_ptr()
    _check_y(y, ref, [x, r], w, 512)
    # a base that is not on 16 bytes: element loads
    y2 = fpkern.add_rms_norm([x.contiguous().view(-1)[1:1 + 39 * 512].view(39, 512)], None, EPS)
    ref2, _ = _ref([x.contiguous().view(-1)[1:1 + 39 * 512].view(39, 512)], None)
    _check_y(y2, ref2, [x.contiguous().view(-1)[1:1 + 39 * 512].view(39, 512)], None, 512)


@pytest.mark.parametrize("off", [1, 2, 5])
@pytest.mark.parametrize("dt", [torch.float16, torch.float32])
def test_bases_off_16_bytes(dt, off):
    """Addends, sum and result at one place within 16 bytes, and at different ones; the elements
    before and behind stay as they were."""
    rows, n = 400, 333
    g = torch.Generator(device="cuda").manual_seed(off)
    bufs = [torch.randn(rows * n + 16, generator=g, device="cuda").to(dt) for _ in range(2)]
    w = torch.randn(n, generator=g, device="cuda").to(dt)
    for offs in ((off, off), (off, off + 1)):
        adds = [b[o:o + rows * n].view(rows, n) for b, o in zip(bufs, offs)]
        ref, s = _ref(adds, w)
        buf = torch.full((rows * n + 16,), 7.0, device="cuda", dtype=dt)
        out = buf[off:off + rows * n].view(rows, n)
        y, total = fpkern.add_rms_norm(adds, w, EPS, return_sum=True, out=out)
        _check_y(y, ref, adds, w, n)
        assert buf[:off].eq(7).all() and buf[off + rows * n:].eq(7).all()
        assert torch.equal(total, (adds[0].float() + adds[1].float()).to(dt))
        q, scale = fpkern.rms_norm_q8(adds, w, EPS)
        _check_q(q, scale, ref, adds, n)


def test_rows_behind_the_last_are_left_and_empty_calls():
    for n in (64, 512, 4096, 40000):
        buf = torch.full((6, n), 7.0, device="cuda")
        fpkern.rms_norm(torch.randn(5, n, device="cuda"), None, EPS, out=buf[:5])
        assert buf[5].eq(7).all()
    q, scale = fpkern.rms_norm_q8([torch.empty(0, 64, device="cuda")], None, EPS)
    assert q.shape == (0, 64) and scale.shape == (0,)


def test_captured_and_replayed():
    x, r = (torch.randn(16, 4096, device="cuda").half() for _ in range(2))
    w = torch.ones(4096, device="cuda").half()
    fpkern.rms_norm_q8([x, r], w, EPS, return_sum=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q, scale, s = fpkern.rms_norm_q8([x, r], w, EPS, return_sum=True)
    for seed in range(3):
        x.copy_(torch.randn(16, 4096, device="cuda"))
        g.replay()
        q2, scale2, s2 = fpkern.rms_norm_q8([x, r], w, EPS, return_sum=True)
        assert torch.equal(q, q2) and torch.equal(scale, scale2) and torch.equal(s, s2)


def test_refusals():
    x = torch.randn(4, 64, device="cuda")
    with pytest.raises(ValueError, match="dtype"):
        fpkern.rms_norm(x.double(), None, EPS)
    with pytest.raises(ValueError, match="one dtype"):
        fpkern.add_rms_norm([x, x.half()], None, EPS)
    with pytest.raises(ValueError, match="shape"):
        fpkern.add_rms_norm([x, x[:, :32]], None, EPS)
    with pytest.raises(ValueError, match="weight"):
        fpkern.rms_norm(x, torch.ones(64, device="cuda").half(), EPS)
    with pytest.raises(ValueError, match="addends"):
        fpkern.add_rms_norm([x] * 5, None, EPS)
    with pytest.raises(ValueError, match="gradient"):
        fpkern.rms_norm(x.clone().requires_grad_(), None, EPS)
    with pytest.raises(ValueError, match="eps"):
        fpkern.rms_norm(x, None, -1.0)
    with pytest.raises(ValueError, match="empty"):
        fpkern.rms_norm(x[:, :0], None, EPS)
    with torch.no_grad():
        fpkern.rms_norm(x.clone().requires_grad_(), None, EPS)
    lib = _lib.load()
    d = _lib.RmsDesc(size=ctypes.sizeof(_lib.RmsDesc), version=_lib.FPK_ABI_VERSION, dtype=_lib.FPK_F32, rows=4,
                     cols=64, q_stride=64, eps=EPS)
    p = ctypes.c_void_p(x.data_ptr())
    a = (ctypes.c_void_p * 1)(x.data_ptr())
    bc = (ctypes.c_int32 * 1)(0)
    call = lambda y, q, s: lib.fpk_rms_norm_fwd(ctypes.byref(d), a, bc, 1, None, None, y, q, s, None)
    assert call(None, None, None) == _lib.FPK_ERR_INVALID  # no output
    assert call(p, p, p) == _lib.FPK_ERR_INVALID           # both
    assert call(None, p, None) == _lib.FPK_ERR_INVALID     # no scale
    d.q_stride = 32
    assert call(None, p, p) == _lib.FPK_ERR_INVALID
    d.cols = 0
    assert call(p, None, None) == _lib.FPK_ERR_INVALID


@pytest.mark.parametrize("rows, n, off", [(5, 40, 0), (7, 512, 0), (400, 1024, 0), (400, 333, 1), (1000, 4096, 0), (9, 9000, 0),
                                          (3, 40000, 0), (3, 5001, 1)])
@pytest.mark.parametrize("place", [0, 1])
def test_out_may_be_an_addend(rows, n, off, place):
    """Every form of the kernel, in the memory of the first or the second addend."""
    g = torch.Generator(device="cuda").manual_seed(n)
    bufs = [torch.randn(rows * n + 8, generator=g, device="cuda") for _ in range(2)]
    adds = [b[off:off + rows * n].view(rows, n) for b in bufs]
    w = torch.randn(n, generator=g, device="cuda")
    want, total = fpkern.add_rms_norm([a.clone() for a in adds], w, EPS, return_sum=True)
    y, kept = fpkern.add_rms_norm(adds, w, EPS, return_sum=True, out=adds[place])
    assert y.data_ptr() == adds[place].data_ptr() and torch.equal(kept, total)
    # another base may run another form, whose sum of squares is in another order (n 2^-24 of it at most)
    torch.testing.assert_close(y, want, atol=1e-6, rtol=n * 2.0 ** -24 + 1e-6)


@pytest.mark.parametrize("n", [1, 33, 127, 129, 319, 321, 639, 641, 1279, 1281, 2559, 2561, 5119, 5121, 8191, 16383, 16385])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
def test_many_rows_of_odd_lengths(dt, n):
    """Rows off 16 bytes around each choice of threads a row: one and two addends, the sum kept, 8 bits."""
    rows = 301
    g = torch.Generator(device="cuda").manual_seed(n)
    x, r = (torch.randn(rows, n, generator=g, device="cuda").to(dt) for _ in range(2))
    w = (1 + 0.1 * torch.randn(n, generator=g, device="cuda")).to(dt)
    for adds in ([x], [x, r]):
        ref, _ = _ref(adds, w)
        y, total = fpkern.add_rms_norm(adds, w, EPS, return_sum=True)
        _check_y(y, ref, adds, w, n)
        assert torch.equal(total, sum(a.float() for a in adds).to(dt))
        q, scale, kept = fpkern.rms_norm_q8(adds, w, EPS, return_sum=True)
        _check_q(q, scale, ref, adds, n)
        assert torch.equal(kept, total)
