"""GPU: what the quantised block's operators make of a tensor's derivative, version and memory."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from fusionpass_b200 import fpkern

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _r(*shape):
    return torch.randn(shape, device=DEV)


def _calls():
    """name -> (operator of its tensors, the tensors, by place, that may carry a derivative)"""
    w, ws = fpkern.quantize_q8(_r(24, 64))
    x, xs = fpkern.quantize_q8(_r(5, 64))
    return {
        "rms_norm": (lambda a, b: fpkern.rms_norm(a, b, 1e-6), [_r(5, 64), _r(64)]),
        "add_rms_norm": (lambda a, b, c: fpkern.add_rms_norm([a, b], c, 1e-6), [_r(5, 64), _r(5, 64), _r(64)]),
        "rms_norm_q8": (lambda a, b: fpkern.rms_norm_q8([a], b, 1e-6), [_r(5, 64), _r(64)]),
        "quantize_q8": (fpkern.quantize_q8, [_r(5, 64)]),
        "linear_q8": (lambda a, b, c: fpkern.linear_q8(x, a, w, b, c, out_dtype=torch.float32), [xs, ws, _r(24)]),
        "score_attention": (lambda a, b, c, d: fpkern.score_attention(a, b, c, 0.1, slopes=d),
                            [_r(1, 2, 5, 64), _r(1, 2, 9, 64), _r(1, 2, 9, 64), _r(2)]),
        "score_attention_f16": (lambda a, b, c, d: fpkern.score_attention(a, b, c, 0.1, slopes=d),
                                [_r(1, 2, 50, 64).half(), _r(1, 2, 90, 64).half(), _r(1, 2, 90, 64).half(), _r(2)]),
    }


@pytest.mark.parametrize("name", ["rms_norm", "add_rms_norm", "rms_norm_q8", "quantize_q8", "linear_q8", "score_attention",
                                  "score_attention_f16"])
def test_a_tangent_is_refused_not_dropped(name):
    f, tensors = _calls()[name]
    want = f(*tensors)
    with fwd.dual_level():
        for i, t in enumerate(tensors):
            dual = fwd.make_dual(t, torch.ones_like(t))
            with pytest.raises(ValueError, match="tangent"):
                f(*tensors[:i], dual, *tensors[i + 1:])
            with torch.inference_mode():  # no derivatives asked for
                f(*tensors[:i], dual, *tensors[i + 1:])
        again = f(*tensors)
    for a, b in zip(want if isinstance(want, tuple) else [want], again if isinstance(again, tuple) else [again]):
        assert torch.equal(a, b)


def test_a_result_with_a_tangent_is_refused():
    x, out = _r(4, 64), _r(4, 64)
    with fwd.dual_level():
        dual = fwd.make_dual(out, torch.ones_like(out))
        with pytest.raises(ValueError, match="tangent"):
            fpkern.rms_norm(x, None, 1e-6, out=dual)


def _outs():
    w, ws = fpkern.quantize_q8(_r(24, 64))
    x, xs = fpkern.quantize_q8(_r(5, 64))
    q, k = _r(1, 2, 5, 64), _r(1, 2, 9, 64)
    a = _r(5, 64)
    return {"rms_norm": ((5, 64), lambda out: fpkern.rms_norm(a, None, 1e-6, out=out)),
            "linear_q8": ((5, 24), lambda out: fpkern.linear_q8(x, xs, w, ws, out_dtype=torch.float32, out=out)),
            "score_attention": ((1, 2, 5, 64), lambda out: fpkern.score_attention(q, k, k, 0.1, out=out))}


@pytest.mark.parametrize("name", ["rms_norm", "linear_q8", "score_attention"])
def test_a_written_result_is_a_new_version(name):
    """What autograd has saved of the memory is known to be gone, as with torch's own results."""
    shape, call = _outs()[name]
    out = _r(*shape)
    leaf = _r(*shape).requires_grad_()
    y = (leaf * out).sum()  # saves out
    before = out._version
    with torch.no_grad():
        call(out)
    assert out._version == before + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    buf = _r(3, *shape)
    view = buf[1]
    before = buf._version
    call(view)
    assert buf._version == before + 1  # a view's base
    with torch.inference_mode():
        held = torch.empty(shape, device=DEV)
    assert torch.equal(call(held), call(None))  # has no version


def test_results_over_an_operand_are_refused():
    buf = _r(4 * 5 * 64).half()
    t = lambda n, *shape: buf[n:n + torch.Size(shape).numel()].view(shape)  # noqa: E731
    x = t(0, 5, 64)
    for call in (lambda: fpkern.rms_norm(x, None, 1e-6, out=t(8, 5, 64)),                      # a part of the addend
                 lambda: fpkern.add_rms_norm([_r(5, 64).half(), t(64, 64)], None, 1e-6, out=x),  # a bias within the result
                 lambda: fpkern.rms_norm(_r(5, 64).half(), t(320 - 64, 64), 1e-6, out=x),       # the weight
                 lambda: fpkern.add_rms_norm([x], None, 1e-6, out=t(64, 5, 64))):
        before = buf.clone()
        with pytest.raises(ValueError, match="overlaps"):
            call()
        assert torch.equal(buf, before)
    w, ws = fpkern.quantize_q8(_r(32, 64))
    q, qs = fpkern.quantize_q8(_r(5, 64))
    bias = t(0, 32)
    for at in (16, 0):
        with pytest.raises(ValueError, match="overlaps"):
            fpkern.linear_q8(q, qs, w, ws, bias, out=t(at, 5, 32))
    with pytest.raises(ValueError, match="overlaps"):  # the activations themselves
        fpkern.linear_q8(q, qs, w, ws, out=q.view(torch.float16))
    q4, k4 = t(0, 1, 2, 5, 64), t(640, 1, 1, 9, 64)
    for out in (q4, t(320, 1, 2, 5, 64), k4.expand(1, 1, 9, 64)[:, :, :5].expand(1, 1, 5, 64)):
        with pytest.raises(ValueError, match="overlaps"):
            fpkern.score_attention(q4[:, :out.shape[1]], k4, k4, 0.1, out=out)


def test_results_beside_their_operands_are_not():
    """In an addend's own memory, behind it, or between the rows of an operand in one buffer."""
    buf = _r(2, 5, 64)
    want = fpkern.rms_norm(buf[0].clone(), None, 1e-6)
    assert torch.equal(fpkern.rms_norm(buf[0], None, 1e-6, out=buf[1]), want)
    row = buf[0, 0].clone()
    want = fpkern.add_rms_norm([row], None, 1e-6, shape=[1, 64])
    assert torch.equal(fpkern.add_rms_norm([row], None, 1e-6, shape=[1, 64], out=row.view(1, 64)), want)  # by its column form
    qkvo = _r(1, 5, 4, 2, 64).half()  # q, k, v and the result of each position side by side
    q, k, v, o = (qkvo[:, :, i].transpose(1, 2) for i in range(4))
    want = fpkern.score_attention(q, k, v, 0.1)
    kept = qkvo[:, :, :3].clone()
    assert torch.equal(fpkern.score_attention(q, k, v, 0.1, out=o), want)
    assert torch.equal(qkvo[:, :, :3], kept)
