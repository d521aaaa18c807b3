"""The quantised block's operators as a model writes them, in plain torch.

``score_attention`` and ``linear_q8`` are ordinary functions (``LinearQ8`` is the module
around the latter) that run anywhere in elementary torch operations; they say what the
operators compute, and a model uses them where ``torch`` has no operator of its own.
``compile_model(..., extensions=True)`` traces each as one plan step, and the plan runtime
runs the step in ``libfpkern.so`` on a CUDA device (``fpkern.score_attention``,
``fpkern.linear_q8``, and ``fpkern.rms_norm_q8`` where the linear reads a norm).
"""

from __future__ import annotations

import torch
from torch import nn
from torch.overrides import handle_torch_function, has_torch_function


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, scale)``: int8 rows and f32 scales, ``scale`` the row's largest magnitude over 127
    (NaN for a row with an infinity or a NaN, and q 0; 0 where that magnitude is below 1.5e-36)."""
    f = x.float()
    top = f.abs().amax(-1)
    ok, some = torch.isfinite(top), top >= 127 * torch.finfo(torch.float32).smallest_normal
    scale = torch.where(ok, torch.where(some, top / 127.0, 0.0), float("nan"))
    q = f / torch.where(ok & some, scale, 1.0).unsqueeze(-1)
    q = torch.where((ok & some).unsqueeze(-1), torch.round(q), 0.0).clamp(-127, 127)
    return q.to(torch.int8), scale


def linear_q8(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
              bias: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ (weight * weight_scale[:, None]).T + bias`` with ``x`` [..., K] (f16 or f32) quantised
    a row at a time, ``weight`` int8 [N, K], ``weight_scale`` f32 [N], ``bias`` of x's dtype; the
    8-bit product is exact and rounded once, to x's dtype, after the scales and the bias."""
    if has_torch_function((x, weight, weight_scale)):
        return handle_torch_function(linear_q8, (x, weight, weight_scale), x, weight, weight_scale, bias)
    q, scale = quantize_rows(x)
    y = (q.double() @ weight.double().transpose(0, 1)) * scale.double().unsqueeze(-1) * weight_scale.double()
    if bias is not None:
        y = y + bias.double()
    return y.to(x.dtype)


class LinearQ8(nn.Module):
    """``nn.Linear`` with an 8-bit weight and a scale an output channel, for inference.  Its
    weight and scale are buffers; ``from_linear`` makes one of an ``nn.Linear``."""

    def __init__(self, weight: torch.Tensor, weight_scale: torch.Tensor, bias: torch.Tensor | None = None):
        super().__init__()
        if weight.dtype != torch.int8 or weight.dim() != 2 or weight_scale.shape != weight.shape[:1]:
            raise ValueError("LinearQ8 needs an int8 weight [N, K] and a scale [N]")
        self.register_buffer("weight", weight)
        self.register_buffer("weight_scale", weight_scale.float())
        self.register_buffer("bias", bias)

    @classmethod
    def from_linear(cls, linear: nn.Linear) -> "LinearQ8":
        with torch.no_grad():
            q, scale = quantize_rows(linear.weight)
            return cls(q, scale, None if linear.bias is None else linear.bias.detach().clone())

    def _apply(self, fn, recurse=True):
        # half() and the like convert the bias; the scales stay in f32, as the operator takes them
        scale = self.weight_scale
        super()._apply(fn, recurse)
        if self.weight_scale.dtype != torch.float32:
            self.weight_scale = scale.to(self.weight_scale.device)
        return self

    def forward(self, x):
        return linear_q8(x, self.weight, self.weight_scale, self.bias)


def score_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, *, softcap: float | None = None,
                    slopes: torch.Tensor | None = None, causal: bool = False, window: int | None = None,
                    prefix: int | torch.Tensor | None = None, doc_ids: torch.Tensor | None = None,
                    kv_lens: torch.Tensor | None = None) -> torch.Tensor:
    """Attention with capped, biased and masked scores over grouped heads; arguments and meaning
    as ``fpkern.score_attention``, in f32 with one rounding of the result."""
    given = tuple(t for t in (q, k, v, slopes, prefix, doc_ids, kv_lens) if t is not None and not isinstance(t, int))
    if has_torch_function(given):
        return handle_torch_function(score_attention, given, q, k, v, scale, softcap=softcap, slopes=slopes,
                                     causal=causal, window=window, prefix=prefix, doc_ids=doc_ids, kv_lens=kv_lens)
    b, h, sq, d = q.shape
    hk, sk = k.shape[1], k.shape[2]
    if sk == 0:
        return torch.zeros_like(q)
    g = h // hk
    lens = kv_lens.long().clamp(0, sk) if kv_lens is not None else torch.full((b,), sk, device=q.device)
    at_q = lens[:, None] - sq + torch.arange(sq, device=q.device)
    at_k = torch.arange(sk, device=q.device)
    ahead = at_k - at_q[:, :, None]
    seen = torch.ones_like(ahead, dtype=torch.bool)
    if causal:
        seen = seen & (ahead <= 0)
    if window is not None:
        seen = seen & (ahead.abs() < window)
    if prefix is not None:
        pre = prefix.long()[:, None, None] if isinstance(prefix, torch.Tensor) else prefix
        seen = seen | (at_k < pre)
    seen = seen & (at_k < lens[:, None, None])
    if doc_ids is not None:
        own = doc_ids.gather(1, at_q.clamp(0, sk - 1))[:, :, None]
        seen = seen & (at_q[:, :, None] >= 0) & (own == doc_ids[:, None, :]) & (own >= 0)
    used = seen.any(1)[:, None, :, None]  # what no query sees may hold anything
    kf, vf = torch.where(used, k.float(), 0.0), torch.where(used, v.float(), 0.0)
    x = (q.float().reshape(b, hk, g * sq, d) @ kf.transpose(-1, -2)).reshape(b, hk, g, sq, sk) * scale
    if softcap is not None:
        x = softcap * torch.tanh(x / softcap)
    if slopes is not None:
        x = x - slopes.float().reshape(1, hk, g, 1, 1) * ahead.abs()[:, None, None].float()
    x = torch.where(seen[:, None, None], x, float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0.0, 1.0, total)
    return (p.reshape(b, hk, g * sq, sk) @ vf).reshape(b, h, sq, d).to(q.dtype)
