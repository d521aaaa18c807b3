"""The bound of score attention's error in f16 and bf16, with every term from the code as it is.

out_i = sum_j w_ij v_j in the notation of _score_ref.py; u = eps/2 of the type.

* a score is off by dx <= D 2^-23 sum_d |scale q_d k_d| (f32 sums of D products on the tensor
  cores, an ulp each) + 4 * 2^-23 max|x| (factor, offset, bias and maximum: each a rounding of a
  value of at most max|x| or |scale q.k|, the difference at most twice that) + 1.1e-6 cap:

  cap tanh(s / cap) = 2 cap y - cap with y = 1 / (1 + e), e = 2^(in s).  In steps of 2^-24 relative
  to y: 1 + e 1; a, a b and r b and their like 1 each, the reciprocal 2 (one ulp), the last product 1;
  the factors b etc. divide out, 1 + 1 + 1 + 2 + 1 + 1 = 7, and 2 cap y 7 <= 14 cap steps.  ex2 is
  within 2^-22 = 4 steps: 2 cap dy <= 2 cap e / (1 + e)^2 4 <= 2 cap steps.  Its argument takes four
  roundings: cap x / cosh^2(x) 4 <= 1.8 cap steps.  17.8 2^-24 = 1.06e-6.
* exponentials are within 2^-22 (ex2.approx), and so are the factors with which parts are joined or
  scaled anew, of which a key meets at most three that its neighbours do not (a new maximum of its
  own, its warp or split, the last joining): e = 4 * 2^-22.  A weight is off by 2 (e + dx), its own
  and the sum's.
* weights are rounded to the type for the product: u, or in f16 below 2^-14 half of 2^-24 while their
  sum is at least 1 (the largest is 2^0 or more): Sk 2^-25 max|v|.
* sums of n keys in f32: n 2^-23; the store rounds by u |out|, the division by 2^-23 |out|."""

import torch

from tests._score_ref import visible

CAP = 17.8 * 2.0 ** -24


def reference(q, k, v, scale, softcap=None, slopes=None, **mask):
    """(out, bound) in 64 bits; k and v are finite."""
    B, H, Sq, D = q.shape
    Hk, Sk = k.shape[1], k.shape[2]
    near, p, j = visible(B, Sq, Sk, device=q.device, **mask)
    near = near[:, None]
    kd, vd, qd = k.double().repeat_interleave(H // Hk, 1), v.double().repeat_interleave(H // Hk, 1), q.double()
    raw = qd @ kd.transpose(-1, -2) * scale
    x = raw if softcap is None else softcap * torch.tanh(raw / softcap)
    if slopes is not None:
        x = x - slopes.double()[None, :, None, None] * (p - j).abs()[:, None].double()
    big = torch.where(near, torch.maximum(x.abs(), raw.abs()), 0.0).amax(-1, keepdim=True)
    terms = torch.where(near, (qd.abs() @ kd.abs().transpose(-1, -2)) * abs(scale), 0.0).amax(-1, keepdim=True)
    x = x.masked_fill(~near, float("-inf"))
    top = x.amax(-1, keepdim=True)
    w = torch.exp(x - torch.where(top == float("-inf"), 0.0, top))
    s = w.sum(-1, keepdim=True)
    w = w / torch.where(s == 0, 1.0, s)
    out, mag = w @ vd, w @ vd.abs()
    u = torch.finfo(q.dtype).eps / 2
    dx = D * 2.0 ** -23 * terms + 4 * 2.0 ** -23 * big + (CAP * softcap if softcap else 0.0)
    bound = (u + 2.0 ** -23) * out.abs() + (u + 2 * (4 * 2.0 ** -22 + dx) + Sk * 2.0 ** -23) * mag
    if q.dtype == torch.float16:
        seen = near.any(-1, keepdim=True)
        bound = bound + torch.where(seen, Sk * 2.0 ** -25, 0.0) * vd.abs().amax((2, 3), keepdim=True)
    fi = torch.finfo(q.dtype)
    return out, bound * (1 + 2 * u) + fi.smallest_normal * fi.eps
