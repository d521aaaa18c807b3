"""Plans of the quantised block (CPU): whole numbers reach only the operands that are read as such."""

import copy

import pytest
import torch
from torch import nn

from fusionpass_b200 import UnsupportedOp, block, compile_model, validate_plan
from tests.block_models import DecoderBlock, QuantHead


class One(nn.Module):
    def __init__(self, f):
        super().__init__()
        self.f = f

    def forward(self, x):
        return self.f(x)


class Two(One):
    def forward(self, x, y):
        return self.f(x, y)


X, IDS, W = torch.randn(4, 16), torch.ones(4, 16, dtype=torch.int32), torch.ones(4, 16, dtype=torch.int8)


@pytest.mark.parametrize("model, args", [
    (Two(lambda x, i: torch.relu(x * i)), (X.half(), IDS)), (Two(lambda x, i: x + i), (X, IDS)),
    (Two(lambda x, i: i + x), (X, W)), (One(torch.exp), (IDS,)), (One(lambda i: i * 2.5), (IDS,)),
    (One(lambda i: torch.softmax(i * 2.5, -1)), (W,))],
    ids=["chain", "add", "add_first", "exp", "scale", "scale_i8"])
def test_whole_numbers_in_other_ops_are_refused_at_tracing(model, args):
    for fuse in (True, False):
        with pytest.raises(UnsupportedOp):
            compile_model(model, args, fuse=fuse, extensions=True, verify=False)


def _plans():
    docs, lens = torch.zeros(2, 5, dtype=torch.int32), torch.full((2,), 5, dtype=torch.int32)
    x = torch.randn(2, 5, 128)
    m = DecoderBlock(2, 5, docs=docs, lens=lens).eval()
    return [compile_model(m, (x,), fuse=fuse, extensions=True, verify=False).plan for fuse in (True, False)] + [
        compile_model(QuantHead().eval(), (torch.randn(3, 96), torch.randn(3, 96)), fuse=True, extensions=True, verify=False).plan]


def test_plans_with_whole_numbers_elsewhere_are_malformed():
    for plan in _plans():
        validate_plan(plan)
        whole = [s["name"] for s in plan["inputs"] if s["dtype"] in ("i8", "i32")]
        assert whole
        places = 0
        for i, st in enumerate(plan["steps"]):
            for k, o in enumerate(st["operands"]):
                if o in whole:
                    places += 1
                    continue
                bad = copy.deepcopy(plan)
                bad["steps"][i]["operands"][k] = whole[0]
                with pytest.raises(ValueError, match=f"operand '{whole[0]}' is"):
                    validate_plan(bad)
        assert places


def test_whole_numbers_pass_through_views_that_copy_nothing():
    class M(nn.Module):
        def forward(self, x, w, s):
            return block.linear_q8(x, w.contiguous(), s)

    c = compile_model(M(), (X, W, torch.ones(4)), fuse=True, extensions=True, verify=False)
    assert [s["op"] for s in c.plan["steps"]] == ["linear_q8"]
