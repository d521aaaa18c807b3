"""Benchmarks and the equivalence gate on plans of the quantised block (CPU parts; the GPU's in
test_gpu_block_bench.py)."""

import torch

from fusionpass_b200 import block, compile_model
from fusionpass_b200.bench import plan_bytes
from tests.block_models import DecoderBlock, QuantHead


def _plan(m, *xs, fuse=True):
    return compile_model(m.eval(), xs, fuse=fuse, extensions=True, verify=False).plan


def test_bytes_of_an_8_bit_linear_behind_a_norm():
    xs = (torch.randn(3, 5, 96), torch.randn(3, 5, 96))
    # two addends, the norm's weight, 40 x 96 bytes, their scales and the bias; the result
    assert plan_bytes(_plan(QuantHead(), *xs)) == 2 * 15 * 96 * 4 + 96 * 4 + 40 * 96 + 40 * 4 * 2 + 15 * 40 * 4


def test_bytes_of_a_kept_sum_and_of_ids():
    B, S, hidden = 2, 7, 128
    docs, lens = torch.zeros(B, S, dtype=torch.int32), torch.full((B,), S, dtype=torch.int32)
    m = DecoderBlock(B, S, docs=docs, lens=lens)
    plan = _plan(m, torch.randn(B, S, hidden))
    step = next(s for s in plan["steps"] if "extra_result" in s)
    row = B * S * 4
    # residual and branch, the norm's weight, the up projection with scales and bias; its result and the sum
    want = 2 * row * hidden + hidden * 4 + 256 * hidden + 2 * 256 * 4 + row * 256 + row * hidden
    assert plan_bytes({**plan, "inputs": plan["inputs"], "steps": [step]} | {
        "inputs": plan["inputs"] + [{"name": o, "shape": [B, S, hidden], "dtype": "f32"} for o in step["operands"]
                                    if o.startswith("v")]}) == want
    att = next(s for s in plan["steps"] if s["op"] == "score_attention")
    heads = [{"name": o, "shape": [B, h, S, 32], "dtype": "f32"} for o, h in zip(att["operands"][:3], (4, 2, 2))]
    assert plan_bytes({**plan, "steps": [att], "inputs": plan["inputs"] + heads}) == (
        row * 32 * (4 + 2 + 2 + 4) + 4 * 4 + B * S * 4 + B * 4)
    assert plan_bytes(plan) < plan_bytes(_plan(m, torch.randn(B, S, hidden), fuse=False))


class _IdsFirst(torch.nn.Module):
    def forward(self, ids, lens, q):
        return block.score_attention(q, q, q, 0.25, causal=True, doc_ids=ids, kv_lens=lens)


class _IdsOnly(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.register_buffer("q", torch.randn(1, 2, 9, 16, generator=torch.Generator().manual_seed(0)))

    def forward(self, ids):
        return block.score_attention(self.q, self.q, self.q, 0.25, doc_ids=ids)


def test_the_gate_takes_its_tolerance_from_the_first_values():
    ids, lens = torch.zeros(1, 9, dtype=torch.int32), torch.full((1,), 9, dtype=torch.int32)
    for dt, tol, name in ((torch.float16, 1e-2, "f16"), (torch.float32, 1e-4, "f32")):
        c = compile_model(_IdsFirst(), (ids, lens, torch.randn(1, 2, 9, 16).to(dt)), extensions=True)
        assert c.verified and (c.report.dtype, c.report.atol, c.report.rtol) == (name, tol, tol)
    assert compile_model(_IdsOnly(), (ids,), extensions=True).report.dtype == "f32"
