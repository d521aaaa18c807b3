"""Plans of the quantised block (CPU): shapes and factors that the plain torch forms stretch or take,
but the operators do not, are refused at tracing instead of in the step on the device."""

import pytest
import torch
import torch.nn.functional as F
from torch import nn

from fusionpass_b200 import UnsupportedOp, block, compile_model


class Call(nn.Module):
    def __init__(self, f, **buffers):
        super().__init__()
        self.f = f
        for name, t in buffers.items():
            self.register_buffer(name, t)

    def forward(self, x):
        return self.f(self, x)


def i32(*shape):
    return torch.ones(shape, dtype=torch.int32)


W = {"w": torch.zeros(8, 16, dtype=torch.int8), "s": torch.ones(8), "one": torch.ones(1), "row": torch.ones(1, 8)}
KV = {"k": torch.randn(1, 2, 7, 16), "k2": torch.randn(2, 2, 7, 16)}


@pytest.mark.parametrize("f, buffers", [
    (lambda m, x: block.linear_q8(x, m.w, m.one), W),
    (lambda m, x: block.linear_q8(x, m.w, m.row), W),
    (lambda m, x: block.linear_q8(x, m.w, m.s, m.one), W),
    (lambda m, x: block.linear_q8(x, m.w, m.s, m.row), W),
    (lambda m, x: block.score_attention(x, x, x, 1.0, prefix=m.p), {"p": i32(1)}),
    (lambda m, x: block.score_attention(x, x, x, 1.0, kv_lens=m.p), {"p": i32(1)}),
    (lambda m, x: block.score_attention(x, m.k, m.k, 1.0), KV),
    (lambda m, x: block.score_attention(x, m.k2, m.k, 1.0), KV),
    (lambda m, x: block.score_attention(x, x, x, 3e38), {}),
    (lambda m, x: block.score_attention(x, x, x, float("inf")), {}),
    (lambda m, x: block.score_attention(x, x, x, float("nan")), {}),
    (lambda m, x: block.score_attention(x, x, x, 1.0, softcap=1e-39), {}),
    (lambda m, x: block.score_attention(x, x, x, 1.0, softcap=1e-50), {}),
    (lambda m, x: block.score_attention(x, x, x, 1.0, softcap=float("nan")), {}),
    (lambda m, x: block.score_attention(x, x, x, 1.0, softcap=float("inf")), {}),
    (lambda m, x: block.score_attention(x, x, x, 1e10, softcap=1e-29), {}),
    (lambda m, x: F.rms_norm(x, (16,), None, -1.0), {})],
    ids=["scale_1", "scale_row", "bias_1", "bias_row", "prefix_1", "lens_1", "batch_of_k_v", "batch_of_v", "scale_large",
         "scale_inf", "scale_nan", "cap_tiny", "cap_zero_in_f32", "cap_nan", "cap_inf", "cap_to_scale", "eps"])
def test_refused_at_tracing(f, buffers):
    x = torch.randn(2, 2, 7, 16)
    for fuse in (True, False):
        with pytest.raises(UnsupportedOp):
            compile_model(Call(f, **buffers), (x,), fuse=fuse, extensions=True, verify=False)


def test_more_columns_than_the_sum_holds():
    w = torch.zeros(2, 131072, dtype=torch.int8)
    f = lambda m, x: block.linear_q8(x, m.w, m.s)  # noqa: E731
    with pytest.raises(UnsupportedOp, match="131071"):
        compile_model(Call(f, w=w, s=torch.ones(2)), (torch.randn(1, 131072),), extensions=True, verify=False)
    c = compile_model(Call(f, w=w[:, :131071].contiguous(), s=torch.ones(2)), (torch.randn(1, 131071),), extensions=True,
                      verify=False)
    assert [s["op"] for s in c.plan["steps"]] == ["linear_q8"]


@pytest.mark.parametrize("kw", [{}, {"softcap": 1e-37}, {"softcap": 1000.0, "window": 1, "prefix": 0},
                                {"slopes": torch.ones(4), "prefix": i32(2), "kv_lens": i32(2), "doc_ids": i32(2, 9)}])
def test_what_the_operator_takes_is_still_traced(kw):
    class M(nn.Module):
        def __init__(self):
            super().__init__()
            for name, t in kw.items():
                if isinstance(t, torch.Tensor):
                    self.register_buffer(name, t)

        def forward(self, q, k):
            return block.score_attention(q, k, k, -0.5, **{n: getattr(self, n) if isinstance(t, torch.Tensor) else t
                                                           for n, t in kw.items()})

    q, k = torch.randn(2, 4, 5, 32), torch.randn(2, 2, 9, 32)
    c = compile_model(M(), (q, k), extensions=True, verify=False)
    assert [s["op"] for s in c.plan["steps"]] == ["score_attention"]
    assert torch.equal(c(q, k), M()(q, k))
