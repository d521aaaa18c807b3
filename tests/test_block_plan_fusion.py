"""Plans of the quantised block (CPU): fusions where one value is read in several places."""

import pytest
import torch
import torch.nn.functional as F
from torch import nn

from fusionpass_b200 import block, compile_model


class Two(nn.Module):
    def __init__(self, f, **buffers):
        super().__init__()
        self.f = f
        for name, t in buffers.items():
            self.register_buffer(name, t)

    def forward(self, x, r):
        return self.f(self, x, r)


def _weighed(m, x, r):
    s = x + r
    return F.rms_norm(s, (16,), s, 1e-6)


def _weighed_and_kept(m, x, r):
    s = x + r
    return F.rms_norm(s, (16,), s, 1e-6) + s


def _weighed_by_an_addend(m, x, r):
    return F.rms_norm(x + r, (16,), r, 1e-6)


def _weighed_linear(m, x, r):
    s = x + r
    return block.linear_q8(F.rms_norm(s, (16,), s, 1e-6), m.w, m.ws)


def _weighed_by_another_norm(m, x, r):
    s = x + r
    return F.rms_norm(s, (16,), F.rms_norm(s, (16,), None, 1e-6), 1e-6)


@pytest.mark.parametrize("f", [_weighed, _weighed_and_kept, _weighed_by_an_addend, _weighed_linear, _weighed_by_another_norm])
def test_a_norm_weighed_by_what_it_sums(f):
    g = torch.Generator().manual_seed(1)
    w = torch.randint(-9, 9, (8, 16), dtype=torch.int8, generator=g)
    xs = tuple(torch.randn(16, generator=g) for _ in range(2))
    m = Two(f, w=w, ws=torch.full((8,), 1e-2)).eval()
    c = compile_model(m, xs, fuse=True, extensions=True, verify=False)
    # one activation off by a step of 1 / 127 of the largest, times a weight of at most 0.09
    torch.testing.assert_close(c(*xs), m(*xs), atol=1e-5 if f is not _weighed_linear else 16 * 0.09 * 2 / 127 * 4, rtol=1e-5)
    named = {i["name"] for i in c.plan["inputs"]}
    for s in c.plan["steps"]:
        assert set(s["operands"]) <= named
        named |= {s["result"], s.get("extra_result", s["result"])}


def _sum_and_norm(m, x, r):
    s = x + r
    return block.linear_q8(s, m.w, m.ws) + F.rms_norm(s, (16,), None, 1e-6)


def _norm_of_sum_unread(m, x, r):
    s = x + r
    F.rms_norm(s, (16,), None, 1e-6)
    return block.linear_q8(s, m.w, m.ws)


@pytest.mark.parametrize("f", [_sum_and_norm, _norm_of_sum_unread])
def test_a_linear_that_reads_the_sum_beside_its_norm(f):
    """The sum is the norm step's second result: the linear quantises the sum, not the norm."""
    g = torch.Generator().manual_seed(2)
    w = torch.randint(-9, 9, (16, 16), dtype=torch.int8, generator=g)
    xs = tuple(3 * torch.randn(4, 16, generator=g) for _ in range(2))
    m = Two(f, w=w, ws=torch.full((16,), 1e-2)).eval()
    c = compile_model(m, xs, fuse=True, extensions=True, verify=False)
    assert [s["op"] for s in c.plan["steps"]][:2] == ["add_rms_norm", "linear_q8"]
    torch.testing.assert_close(c(*xs), m(*xs), atol=1e-5, rtol=1e-5)
