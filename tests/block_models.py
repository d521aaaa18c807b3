"""Blocks with the quantised operators, as a model would write them."""

import torch
import torch.nn.functional as F
from torch import nn

from fusionpass_b200 import LinearQ8, score_attention


class DecoderBlock(nn.Module):
    """Pre-norm block: RMS norms, 8-bit projections, grouped heads with capped and biased causal
    scores over documents."""

    def __init__(self, batch, seq, hidden=128, heads=4, kv_heads=2, ffn=256, docs=None, lens=None, seed=0):
        super().__init__()
        self.B, self.S, self.H, self.Hk, self.D = batch, seq, heads, kv_heads, hidden // heads
        g = torch.Generator().manual_seed(seed)

        def linear(i, o, bias=False):
            m = nn.Linear(i, o, bias=bias)
            with torch.no_grad():
                m.weight.copy_(torch.randn(o, i, generator=g) * i ** -0.5)
                if bias:
                    m.bias.copy_(torch.randn(o, generator=g) * 0.1)
            return LinearQ8.from_linear(m)

        self.n1, self.n2 = nn.RMSNorm(hidden, eps=1e-6), nn.RMSNorm(hidden, eps=1e-6)
        with torch.no_grad():
            self.n1.weight.copy_(1 + 0.1 * torch.randn(hidden, generator=g))
        self.q, self.k, self.v = linear(hidden, hidden), linear(hidden, kv_heads * self.D), linear(hidden, kv_heads * self.D)
        self.o, self.up, self.down = linear(hidden, hidden), linear(hidden, ffn, True), linear(ffn, hidden)
        self.register_buffer("slopes", 2.0 ** (-8.0 * torch.arange(1, heads + 1) / heads))
        self.register_buffer("docs", docs)
        self.register_buffer("lens", lens)

    def half_weights(self):
        """Norm weights and biases in f16; scales and slopes stay in f32."""
        for m in self.modules():
            if isinstance(m, nn.RMSNorm):
                m.half()
            if isinstance(m, LinearQ8) and m.bias is not None:
                m.bias = m.bias.half()
        return self

    def forward(self, x):
        B, S, D = self.B, self.S, self.D
        n = self.n1(x)
        q = self.q(n).view(B, S, self.H, D).transpose(1, 2)
        k = self.k(n).view(B, S, self.Hk, D).transpose(1, 2)
        v = self.v(n).view(B, S, self.Hk, D).transpose(1, 2)
        a = score_attention(q, k, v, D ** -0.5, softcap=20.0, slopes=self.slopes, causal=True, doc_ids=self.docs,
                            kv_lens=self.lens)
        h = x + self.o(a.transpose(1, 2).reshape(B, S, self.H * D))
        return h + self.down(F.gelu(self.up(self.n2(h))))


class QuantHead(nn.Module):
    """A sum's norm that one 8-bit linear reads, and nothing else."""

    def __init__(self, hidden=96, out=40):
        super().__init__()
        g = torch.Generator().manual_seed(1)
        self.norm = nn.RMSNorm(hidden, eps=1e-5)
        w = nn.Linear(hidden, out)
        with torch.no_grad():
            w.weight.copy_(torch.randn(out, hidden, generator=g) * hidden ** -0.5)
        self.lin = LinearQ8.from_linear(w)

    def forward(self, x, r):
        return self.lin(self.norm(x + r))
