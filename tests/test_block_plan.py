"""Plans of the quantised block (CPU): what is traced, fused, validated and refused, and that
the plan's steps compute what the model does."""

import copy
import json

import pytest
import torch
import torch.nn.functional as F
from torch import nn

from fusionpass_b200 import LinearQ8, UnsupportedOp, block, compile_model, execute_plan, validate_plan
from tests._score_ref import close, reference
from tests.block_models import DecoderBlock, QuantHead


def kinds(c):
    return [s.get("launch", s.get("op")) for s in c.plan["steps"]]


def _docs(B, S):
    return (torch.arange(S) * 3 // S).to(torch.int32).expand(B, S).contiguous()


def test_unfused_decoder_block_on_the_cpu():
    B, S = 2, 20
    m = DecoderBlock(B, S, docs=_docs(B, S)).eval()
    x = torch.randn(B, S, 128, generator=torch.Generator().manual_seed(0))
    c = compile_model(m, (x,), fuse=False, extensions=True, verify=False)
    k = kinds(c)
    assert k.count("linear_q8") == 6 and k.count("rms_norm") == 2 and k.count("score_attention") == 1
    # the same steps in the same order; RMS norm sums in another order than torch's
    torch.testing.assert_close(c(x), m(x), atol=5e-3, rtol=5e-3)
    plan = json.loads(json.dumps(c.plan))
    validate_plan(plan)
    assert {i["dtype"] for i in plan["inputs"]} == {"f32", "i8", "i32"}
    assert torch.equal(execute_plan(plan, [x] + c._captured), c(x))


def test_fused_steps_of_the_decoder_block():
    B, S = 1, 16
    m = DecoderBlock(B, S).eval()
    c = compile_model(m, (torch.randn(B, S, 128),), fuse=True, extensions=True, verify=False)
    steps = c.plan["steps"]
    fused = [s for s in steps if s.get("op") == "rms_norm_linear_q8"]
    # the second norm: residual + branch in, sum kept for the residual that goes on, the up projection out
    assert len(fused) == 1 and fused[0]["attrs"]["n_addends"] == 2 and fused[0]["attrs"]["affine"]
    kept = fused[0]["extra_result"]
    assert kept in steps[-1]["operands"]
    # the first norm feeds three projections: a step of its own
    assert kinds(c).count("rms_norm") == 1 and kinds(c).count("linear_q8") == 5
    att = next(s for s in steps if s.get("op") == "score_attention")
    assert att["attrs"]["optional"] == ["slopes"] and att["attrs"]["out_layout"] == [0, 2, 1, 3]
    assert att["attrs"]["softcap"] == 20.0 and att["attrs"]["causal"] is True


def test_fused_head_on_the_cpu():
    m = QuantHead().eval()
    xs = tuple(torch.randn(3, 5, 96, generator=torch.Generator().manual_seed(i)) for i in range(2))
    c = compile_model(m, xs, fuse=True, extensions=True, verify=False)
    assert kinds(c) == ["rms_norm_linear_q8"]
    torch.testing.assert_close(c(*xs), m(*xs), atol=5e-3, rtol=5e-3)


def test_sum_kept_as_an_output_and_norm_read_twice():
    class Kept(nn.Module):
        def __init__(self):
            super().__init__()
            self.norm = nn.RMSNorm(32, eps=1e-6, elementwise_affine=False)

        def forward(self, x, r):
            s = x + r
            n = self.norm(s)
            return torch.relu(n) + s * 2.0

    xs = (torch.randn(4, 32), torch.randn(4, 32))
    g = compile_model(Kept(), xs, fuse=True, extensions=True, verify=False).plan
    assert g["steps"][0]["op"] == "add_rms_norm" and "extra_result" in g["steps"][0]
    assert not g["steps"][0]["attrs"]["affine"]


def test_linear_whose_bias_is_the_kept_sum():
    """The sum is that very step's second result, so the step cannot read it."""
    w, s = torch.randint(-9, 9, (32, 32), dtype=torch.int8, generator=torch.Generator().manual_seed(6)), torch.full((32,), 1e-3)

    class M(nn.Module):
        def __init__(self):
            super().__init__()
            self.norm = nn.RMSNorm(32, eps=1e-6)
            self.register_buffer("w", w)
            self.register_buffer("s", s)

        def forward(self, x, r):
            t = x + r
            return block.linear_q8(self.norm(t), self.w, self.s, t)

    xs = (torch.randn(32, generator=torch.Generator().manual_seed(7)), torch.randn(32, generator=torch.Generator().manual_seed(8)))
    m = M().eval()
    c = compile_model(m, xs, fuse=True, extensions=True, verify=False)
    assert kinds(c) == ["add_rms_norm", "linear_q8"]
    torch.testing.assert_close(c(*xs), m(*xs), atol=5e-3, rtol=5e-3)


def test_functional_rms_norm_and_bias_chain():
    class M(nn.Module):
        def __init__(self):
            super().__init__()
            self.w, self.b = nn.Parameter(torch.rand(24)), nn.Parameter(torch.rand(24))

        def forward(self, x, r):
            return F.rms_norm(x + self.b + r, (24,), self.w, 1e-6)

    xs = (torch.randn(2, 3, 24), torch.randn(2, 3, 24))
    m = M()
    c = compile_model(m, xs, fuse=True, extensions=True, verify=False)
    assert kinds(c) == ["add_rms_norm"] and c.plan["steps"][0]["attrs"]["n_addends"] == 3
    torch.testing.assert_close(c(*xs), m(*xs), atol=1e-5, rtol=1e-5)


def test_default_eps_is_torchs():
    m = nn.Sequential(nn.RMSNorm(16))
    c = compile_model(m, (torch.randn(2, 16),), fuse=True, extensions=True, verify=False)
    assert c.plan["steps"][0]["attrs"]["eps"] == torch.finfo(torch.float32).eps


def test_default_eps_of_f16_is_that_of_f32():
    """Rows whose mean square lies between the two types' epsilons show which one is taken."""
    x = torch.full((3, 16), 1e-3, dtype=torch.float16)

    class M(nn.Module):
        def forward(self, x):
            return F.rms_norm(x, (16,))

    for m in (nn.Sequential(nn.RMSNorm(16).half()), M()):
        c = compile_model(m, (x,), fuse=True, extensions=True, verify=False)
        want = m(x).detach()
        assert want[0, 0] > 0.9
        torch.testing.assert_close(c(x), want, atol=0, rtol=2 * torch.finfo(torch.float16).eps)


def test_without_extensions_nothing_new_is_traced():
    with pytest.raises(UnsupportedOp):
        compile_model(nn.Sequential(nn.RMSNorm(16)), (torch.randn(2, 16),))

    class M(nn.Module):
        def forward(self, q):
            return block.score_attention(q, q, q, 1.0)

    with pytest.raises(UnsupportedOp):
        compile_model(M(), (torch.randn(1, 1, 4, 16),))
    with pytest.raises(UnsupportedOp):
        compile_model(nn.Sequential(nn.RMSNorm((4, 16))), (torch.randn(2, 4, 16),), extensions=True)


def _plan():
    m = QuantHead().eval()
    xs = (torch.randn(3, 96), torch.randn(3, 96))
    return compile_model(m, xs, fuse=True, extensions=True, verify=False).plan


@pytest.mark.parametrize("break_it", [
    lambda s: s["attrs"].update(n_addends=9), lambda s: s["attrs"].update(n_addends=4),
    lambda s: s["attrs"].update(affine=False), lambda s: s["attrs"].update(eps=-1.0),
    lambda s: s.update(extra_result=s["result"]), lambda s: s.update(op="linear_q8"),
    lambda s: s.update(op="rms_norm"), lambda s: s.update(op="score_attention"),
    lambda s: s.update(op="add_rms_norm")])
def test_malformed_steps_are_refused(break_it):
    plan = _plan()
    validate_plan(plan)
    bad = copy.deepcopy(plan)
    break_it(bad["steps"][0])
    with pytest.raises(ValueError):
        validate_plan(bad)


def test_only_norm_steps_have_a_second_result():
    bad = copy.deepcopy(_plan())
    bad["steps"][0].update(op="gelu", extra_result="more")
    with pytest.raises(ValueError, match="second result"):
        validate_plan(bad)


def test_eager_score_attention_is_the_definition():
    g = torch.Generator().manual_seed(3)
    q, k, v = torch.randn(2, 4, 9, 16, generator=g), torch.randn(2, 2, 21, 16, generator=g), torch.randn(2, 2, 21, 16, generator=g)
    kw = {"softcap": 3.0, "slopes": torch.rand(4, generator=g), "causal": True, "window": 6, "prefix": torch.tensor([2, 7]),
          "doc_ids": torch.randint(-1, 2, (2, 21), generator=g).to(torch.int32), "kv_lens": torch.tensor([5, 21], dtype=torch.int32)}
    v[0, :, 6:] = float("nan")  # behind the first sequence's keys
    ref, bound = reference(q, k, v, 0.25, **kw)
    close(block.score_attention(q, k, v, 0.25, **kw), ref, bound)


def test_eager_score_attention_without_keys():
    q, k = torch.randn(2, 4, 3, 16), torch.randn(2, 2, 0, 16)
    for kw in ({}, {"causal": True, "doc_ids": torch.zeros(2, 0, dtype=torch.int32), "prefix": 3, "softcap": 2.0}):
        assert torch.equal(block.score_attention(q, k, k, 0.25, **kw), torch.zeros_like(q))


def test_eager_linear_q8():
    g = torch.Generator().manual_seed(4)
    lin = nn.Linear(50, 30)
    m = LinearQ8.from_linear(lin)
    x = torch.randn(3, 50, generator=g)
    # half a step of each weight and activation
    w = m.weight.double() * m.weight_scale.double()[:, None]
    step_x = x.abs().amax(-1, keepdim=True) / 127
    room = 0.501 * (step_x * w.abs().sum(1) + x.abs().sum(-1, keepdim=True) * m.weight_scale) + 1e-6
    assert ((m(x).double() - lin(x).double()).abs() <= room).all()
    q, s = block.quantize_rows(torch.tensor([[0.0, 0.0], [1.0, float("inf")], [1e-40, 0.0], [-2.0, 1.0]]))
    assert s[0] == 0 and torch.isnan(s[1]) and s[2] == 0 and q[:3].eq(0).all() and q[3].tolist() == [-127, 64]
    with pytest.raises(ValueError):
        LinearQ8(torch.zeros(2, 3), torch.ones(2))


def test_converted_linear_q8_keeps_its_scales():
    m = LinearQ8.from_linear(nn.Linear(32, 8))
    scale = m.weight_scale.clone()
    for convert in (nn.Module.half, nn.Module.double, nn.Module.float, lambda m: m.to(torch.float16)):
        m = convert(m)
        assert m.weight.dtype == torch.int8 and m.weight_scale.dtype == torch.float32
        assert torch.equal(m.weight_scale, scale)
    assert m.bias.dtype == torch.float16 and set(m.state_dict()) == {"weight", "weight_scale", "bias"}
    x = torch.randn(3, 32, generator=torch.Generator().manual_seed(5)).half()
    c = compile_model(nn.Sequential(m), (x,), fuse=True, extensions=True, verify=False)
    assert torch.equal(c(x), m(x))


class _Call(nn.Module):
    def __init__(self, f, **buffers):
        super().__init__()
        self.f = f
        for name, t in buffers.items():
            self.register_buffer(name, t)

    def forward(self, x):
        return self.f(self, x)


_W = {"w": torch.zeros(8, 16, dtype=torch.int8), "s": torch.ones(8), "h": torch.ones(8, dtype=torch.float16)}


@pytest.mark.parametrize("f, buffers, half", [
    (lambda m, x: block.linear_q8(x, m.w, m.h), _W, False),
    (lambda m, x: block.linear_q8(x, m.w, m.s, m.h), _W, False),
    (lambda m, x: block.linear_q8(x, m.g, m.s), {**_W, "g": torch.zeros(8, 16)}, False),
    (lambda m, x: block.score_attention(x, x, x, 1.0, slopes=m.h), {"h": torch.ones(2, dtype=torch.float16)}, False),
    (lambda m, x: block.score_attention(x, x, x, 1.0, softcap=2000.0), {}, True),
    (lambda m, x: block.score_attention(x, x, x, 1.0, softcap=-1.0), {}, False),
    (lambda m, x: block.score_attention(x, x, x, 1.0, window=0), {}, False),
    (lambda m, x: block.score_attention(x, x, x, 1.0, prefix=-1), {}, False),
    (lambda m, x: block.score_attention(*[x.reshape(1, 2, 8, 8)] * 3, 1.0), {}, False),
    (lambda m, x: block.score_attention(x, m.k, m.k, 1.0), {"k": torch.ones(1, 2, 4, 16, dtype=torch.float16)}, False)])
def test_what_the_operators_do_not_take_is_refused_at_tracing(f, buffers, half):
    x = torch.randn(1, 2, 4, 16)
    with pytest.raises(UnsupportedOp):
        compile_model(_Call(f, **buffers), (x.half() if half else x,), fuse=True, extensions=True, verify=False)
