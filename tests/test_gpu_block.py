"""GPU: plans of the quantised block run in libfpkern.so, one behind the other, and agree
with the model's own (plain torch) forms within the compile gate."""

import pytest
import torch

from fusionpass_b200 import block, compile_model, fpkern
from fusionpass_b200.runtime import execute_plan
from tests.block_models import DecoderBlock, QuantHead

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _device_status_clean():
    yield
    assert fpkern.poll_status() == 0


def _spy(monkeypatch):
    calls = []
    for name in ("add_rms_norm", "rms_norm_q8", "quantize_q8", "linear_q8", "score_attention"):
        real = getattr(fpkern, name)
        monkeypatch.setattr(fpkern, name, lambda *a, _n=name, _r=real, **k: (calls.append(_n), _r(*a, **k))[1])
    return calls


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("B,S,hidden,heads,kv,ffn", [(2, 33, 128, 4, 2, 256), (1, 200, 256, 8, 2, 512), (3, 1, 128, 2, 1, 320)])
def test_decoder_block_compiles_and_agrees(monkeypatch, half, B, S, hidden, heads, kv, ffn):
    docs = (torch.arange(S) * 3 // max(S, 1)).to(torch.int32).expand(B, S).contiguous()
    lens = torch.randint(1, S + 1, (B,), generator=torch.Generator().manual_seed(S)).to(torch.int32)
    m = DecoderBlock(B, S, hidden, heads, kv, ffn, docs, lens).eval()
    m = (m.half_weights() if half else m).to(DEV)
    x = torch.randn(B, S, hidden, generator=torch.Generator().manual_seed(1)).to(DEV)
    x = x.half() if half else x
    calls = _spy(monkeypatch)
    # the fused norm quantises its unrounded output, the model its rounded one: a value moves by a
    # step now and then.  A step is max|y| / 127 <= 5 / 127 for a normalised row, a weight about
    # hidden^-1/2; with one in fifty of the values of a row off by one in f16 (rounding moves a
    # value by 2^-12 of its 127 steps at most, 0.03 of a step) the product moves by
    # sqrt(1 / 50) * 5 / 127 = 5.6e-3 (1 sigma) in each of the block's two residual branches:
    # four sigma of both, 0.032
    c = compile_model(m, (x,), fuse=True, extensions=True, atol=0.032, rtol=1e-2)
    assert c.verified
    assert calls.count("score_attention") == 3 and calls.count("rms_norm_q8") == 3
    assert calls.count("linear_q8") == 3 * 6 and calls.count("quantize_q8") == 3 * 5
    y = c(x)
    assert y.shape == x.shape and y.dtype == x.dtype


def test_fused_head_in_one_norm_and_one_product(monkeypatch):
    m = QuantHead(hidden=1000, out=333).eval().to(DEV)
    xs = (torch.randn(70, 1000, device=DEV), torch.randn(70, 1000, device=DEV))
    calls = _spy(monkeypatch)
    c = compile_model(m, xs, fuse=True, extensions=True, verify=False)
    y = c(*xs)
    assert calls == ["rms_norm_q8", "linear_q8"]
    # off by steps of single activations: 1 / 127 of the row's largest, times a weight
    torch.testing.assert_close(y, m(*xs), atol=5 / 127 * 4 * 1000 ** -0.5, rtol=1e-3)


def test_plan_captured_and_replayed():
    B, S = 2, 40
    m = DecoderBlock(B, S).eval().half_weights().to(DEV)
    x = torch.randn(B, S, 128, device=DEV).half()
    c = compile_model(m, (x,), fuse=True, extensions=True, verify=False)
    c(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c(x)  # warm up the compiled chains
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = c(x)
    for seed in range(3):
        x.copy_(torch.randn(B, S, 128, generator=torch.Generator().manual_seed(seed)))
        g.replay()
        torch.testing.assert_close(y, c(x), atol=0.0, rtol=0.0)


def test_ids_and_lengths_as_inputs_of_the_plan():
    class M(torch.nn.Module):
        def forward(self, q, k, v, ids, lens, pre):
            return block.score_attention(q, k, v, 0.125, causal=True, window=50, prefix=pre, doc_ids=ids, kv_lens=lens)

    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(2, h, s, 64, generator=g).half().to(DEV) for h, s in ((4, 60), (2, 130), (2, 130)))
    ids = (torch.arange(130) // 45).to(torch.int32).expand(2, 130).contiguous().to(DEV)
    lens, pre = torch.tensor([100, 130], dtype=torch.int32, device=DEV), torch.tensor([5, 0], dtype=torch.int32, device=DEV)
    m = M()
    c = compile_model(m, (q, k, v, ids, lens, pre), fuse=True, extensions=True)
    assert c.verified
    bad = [q, k, v, ids.long(), lens, pre]
    with pytest.raises(ValueError, match="expected"):
        execute_plan(c.plan, bad, c.kernels)


def test_default_eps_of_f16_is_torchs_on_the_device():
    x = torch.full((300, 64), 1e-3, dtype=torch.float16, device="cuda")
    m = torch.nn.Sequential(torch.nn.RMSNorm(64).half().cuda())
    c = compile_model(m, (x,), fuse=True, extensions=True, verify=False)
    want = m(x).detach()
    torch.testing.assert_close(c(x), want, atol=0, rtol=2 * torch.finfo(torch.float16).eps)


def test_model_halved_as_a_whole():
    m = QuantHead().eval().half().cuda()
    xs = tuple(torch.randn(9, 96, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i)).half() for i in range(2))
    c = compile_model(m, xs, fuse=True, extensions=True, verify=False)
    assert m.lin.weight_scale.dtype == torch.float32
    # four sigma of one in fifty activations off by a step, as in the decoder block, and a rounding
    torch.testing.assert_close(c(*xs), m(*xs), atol=0.0224, rtol=2.0 ** -10)
