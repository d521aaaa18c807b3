"""GPU: the 8-bit linear against the formula in 64 bits.

The integer sum is exact, so with scales and bias in f32 the result before the store is
off by 3 roundings of the product (sum to f32, two scales) and one of the addition: with
u = eps/2 of the output type, |y - ref| <= u |ref| + 4 * 2^-24 * (|product| + |bias|)."""

import ctypes

import pytest
import torch

from fusionpass_b200 import _lib, fpkern

pytestmark = pytest.mark.gpu


def _inputs(m, n, k, dt, seed, bias=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randint(-128, 128, (m, k), generator=g, device="cuda").to(torch.int8)
    w = torch.randint(-128, 128, (n, k), generator=g, device="cuda").to(torch.int8)
    xs = torch.rand(m, generator=g, device="cuda") * 0.05
    ws = torch.rand(n, generator=g, device="cuda") / (70.0 * 70.0 * 0.05)
    b = torch.randn(n, generator=g, device="cuda").to(dt) if bias else None
    return x, xs, w, ws, b


def _check(y, x, xs, w, ws, b):
    prod = (x.double() @ w.double().T) * xs.double()[..., None] * ws.double()
    add = b.double() if b is not None else torch.zeros((), device="cuda", dtype=torch.float64)
    ref = prod + add
    fi = torch.finfo(y.dtype)
    room = fi.eps / 2 * (1 + 1e-3) * ref.abs() + 4 * 2.0 ** -24 * (prod.abs() + add.abs()) + fi.smallest_normal * fi.eps
    sat = ref.abs() > fi.max * (1 - fi.eps)  # f16 overflows to infinity, as the rounding of the value does
    assert ((y.double() - ref).abs() <= room)[~sat].all()


# token tiles of 16, 32, 64, 128 and 256 and around their borders; channels and K around a tile; K shared
# by 1, 2, 4 and 8 CTAs; more tiles than SMs
SIZES = [(1, 1, 1), (1, 128, 128), (7, 130, 100), (16, 64, 4096), (17, 1000, 2048), (33, 300, 1030), (64, 1024, 512),
         (65, 257, 1100), (128, 4096, 1024), (129, 4096, 384), (200, 333, 1001), (333, 1001, 1030),
         (1024, 4096, 640), (1300, 9000, 136), (3, 40000, 256)]


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear_q8(m, n, k, dt):
    x, xs, w, ws, b = _inputs(m, n, k, dt, m + n + k)
    for bias in (b, None):
        y = fpkern.linear_q8(x, xs, w, ws, bias, out_dtype=dt)
        assert y.shape == (m, n) and y.dtype == dt
        _check(y, x, xs, w, ws, bias)
    assert fpkern.poll_status() == 0


def test_sum_at_the_ends_of_32_bits():
    """Every product 2^14 over the longest K: the sum is 131071 * 16384 = 2^31 - 16384."""
    k = _lib.FPK_LINEAR_MAX_K
    x = torch.full((3, k), -128, device="cuda", dtype=torch.int8)
    w = torch.full((130, k), -128, device="cuda", dtype=torch.int8)
    w[1::2] = 127
    y = fpkern.linear_q8(x, torch.ones(3, device="cuda"), w, torch.ones(130, device="cuda"), out_dtype=torch.float32)
    want = torch.full((130,), 16384.0 * k, device="cuda", dtype=torch.float64)
    want[1::2] = -128.0 * 127.0 * k
    assert torch.equal(y, want.float().expand(3, 130))


@pytest.mark.parametrize("m", [1, 40, 300])
def test_strided_padded_and_batched_operands(m):
    x, xs, w, ws, b = _inputs(2 * m, 200, 1030, torch.float16, m)
    ref = fpkern.linear_q8(x, xs, w, ws, b)
    _check(ref, x, xs, w, ws, b)
    xb = x.view(2, m, 1030)
    assert torch.equal(fpkern.linear_q8(xb, xs.view(2, m), w, ws, b), ref.view(2, m, 200))
    padded = torch.full((2 * m, 1040), 99, device="cuda", dtype=torch.int8)
    padded[:, :1030] = x
    assert torch.equal(fpkern.linear_q8(padded[:, :1030], xs, w, ws, b), ref)      # read in place
    assert torch.equal(fpkern.linear_q8(x.T.contiguous().T, xs, w, ws, b), ref)    # copied
    assert torch.equal(fpkern.linear_q8(x, xs.repeat(2)[: 2 * m], w.T.contiguous().T, ws, b), ref)
    # rows that share memory: an expanded row and batch, windows that overlap
    one = x[:1].expand(6, 1030)
    close = fpkern.linear_q8(one, xs[:1].expand(6), w, ws, b)
    assert torch.equal(close, ref[:1].expand(6, 200))
    assert torch.equal(fpkern.linear_q8(x[:1].expand(3, 2, 1030), xs[:1].expand(3, 2), w, ws, b), ref[:1].expand(3, 2, 200))
    assert torch.equal(fpkern.linear_q8(x[None].expand(3, 2 * m, 1030), xs.expand(3, 2 * m), w, ws, b),
                       ref.expand(3, 2 * m, 200))
    flat = x.reshape(-1)
    if flat.numel() >= 1030 + 16 * 4:
        over = flat.as_strided((5, 1030), (16, 1))
        assert torch.equal(fpkern.linear_q8(over, xs[:1].expand(5), w, ws, b),
                           fpkern.linear_q8(over.contiguous(), xs[:1].expand(5), w, ws, b))
    assert torch.equal(fpkern.linear_q8(x, xs, w[:1].expand(200, 1030), ws, b),
                       fpkern.linear_q8(x, xs, w[:1].repeat(200, 1), ws, b))
    odd = torch.empty(2 * m * 1040 + 1, device="cuda", dtype=torch.int8)[1:].view(2 * m, 1040)
    odd[:, :1030] = x
    assert torch.equal(fpkern.linear_q8(odd[:, :1030], xs, w, ws, b), ref)         # base off 16 bytes
    t = xb.transpose(0, 1)
    assert torch.equal(fpkern.linear_q8(t, xs.view(2, m).T, w, ws, b), ref.view(2, m, 200).transpose(0, 1))


def test_scales_of_nan_zero_and_infinity_stay_in_their_rows():
    x, xs, w, ws, _ = _inputs(40, 150, 256, torch.float32, 5)
    xs[3], xs[4] = float("nan"), 0.0
    ws[7] = float("inf")
    y = fpkern.linear_q8(x, xs, w, ws, out_dtype=torch.float32)
    ok = torch.ones(40, 150, dtype=torch.bool, device="cuda")
    ok[3] = False
    ok[:, 7] = False
    assert torch.isnan(y[3]).all() and torch.isfinite(y[ok]).all() and not torch.isfinite(y[:, 7]).any()
    assert y[4][torch.arange(150, device="cuda") != 7].eq(0).all()


def test_out_rows_behind_the_last_stay_and_empty_calls():
    for m in (5, 70, 300):
        x, xs, w, ws, b = _inputs(m, 200, 256, torch.float16, m)
        buf = torch.full((m + 3, 200), 7.0, device="cuda", dtype=torch.float16)
        y = fpkern.linear_q8(x, xs, w, ws, b, out=buf[:m])
        assert y.data_ptr() == buf.data_ptr() and buf[m:].eq(7).all()
        _check(y, x, xs, w, ws, b)
    assert fpkern.linear_q8(x[:0], xs[:0], w, ws).shape == (0, 200)
    assert fpkern.linear_q8(x, xs, w[:0], ws[:0]).shape == (m, 0)


def test_captured_on_a_side_stream_two_graphs():
    """Two captured calls replayed together on two streams."""
    args = [_inputs(m, 1024, 2048, torch.float16, m) for m in (4, 300)]
    graphs, outs = [], []
    for x, xs, w, ws, b in args:
        fpkern.linear_q8(x, xs, w, ws, b)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(fpkern.linear_q8(x, xs, w, ws, b))
        graphs.append(g)
    side = torch.cuda.Stream()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.current_stream().wait_stream(side)
    for y, (x, xs, w, ws, b) in zip(outs, args):
        _check(y, x, xs, w, ws, b)
    assert fpkern.poll_status() == 0


def test_norm_into_linear():
    """The two together, as a block uses them: the product of the 8-bit norm stays within what
    half a step of each activation allows (1-norm of the weights times half a step)."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x, r = (torch.randn(50, 1030, generator=g, device="cuda").half() for _ in range(2))
    nw = torch.ones(1030, device="cuda").half()
    wf = torch.randn(300, 1030, generator=g, device="cuda") * 0.03
    wq, ws = fpkern.quantize_q8(wf)
    q, qs, s = fpkern.rms_norm_q8([x, r], nw, 1e-6, return_sum=True)
    y = fpkern.linear_q8(q, qs, wq, ws, out_dtype=torch.float32)
    _check(y, q, qs, wq, ws, None)
    total = x.double() + r.double()
    norm = total * (total.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    ref = norm @ wf.double().T
    w1 = (wq.double() * ws.double()[:, None]).abs().sum(1)
    room = 0.501 * qs.double()[:, None] * w1 + (norm.abs().sum(1)[:, None]) * 0.501 * ws.double()
    assert ((y.double() - ref).abs() <= room).all()


def test_refusals():
    x, xs, w, ws, b = _inputs(4, 64, 128, torch.float16, 1)
    with pytest.raises(ValueError, match="int8"):
        fpkern.linear_q8(x.half(), xs, w, ws)
    with pytest.raises(ValueError, match="columns"):
        fpkern.linear_q8(x, xs, w[:, :64], ws)
    with pytest.raises(ValueError, match="x_scale"):
        fpkern.linear_q8(x, xs[:3], w, ws)
    with pytest.raises(ValueError, match="w_scale"):
        fpkern.linear_q8(x, xs, w, ws.half())
    with pytest.raises(ValueError, match="bias"):
        fpkern.linear_q8(x, xs, w, ws, b.float())
    with pytest.raises(ValueError, match="dtype"):
        fpkern.linear_q8(x, xs, w, ws, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="out"):
        fpkern.linear_q8(x, xs, w, ws, out=torch.empty(4, 63, device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError, match="K must be"):
        big = torch.zeros(1, _lib.FPK_LINEAR_MAX_K + 1, device="cuda", dtype=torch.int8)
        fpkern.linear_q8(big, xs[:1], big, ws[:1])
    with pytest.raises(RuntimeError, match="CUDA"):
        fpkern.linear_q8(x.cpu(), xs, w, ws)
    lib = _lib.load()
    d = _lib.LinearDesc(size=ctypes.sizeof(_lib.LinearDesc), version=_lib.FPK_ABI_VERSION, out_dtype=_lib.FPK_F16,
                        m=4, n=64, k=100, x_stride=100, w_stride=112, y_stride=64)
    p = ctypes.c_void_p(x.data_ptr())
    call = lambda: lib.fpk_linear_int_fwd(ctypes.byref(d), p, p, p, p, None, p, None, 0, None)
    assert lib.fpk_linear_int_workspace(ctypes.byref(d), p, p) == 4 * 112 + (256 - 4 * 112 % 256)
    assert call() == _lib.FPK_ERR_INVALID  # the workspace for x's rows is missing
    d.x_stride = 96
    assert call() == _lib.FPK_ERR_INVALID
    d.x_stride, d.k = 112, 0
    assert call() == _lib.FPK_ERR_INVALID
