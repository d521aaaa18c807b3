"""Score attention from its definition in 64 bits, and the bound of a kernel's error.

out_i = sum_j w_ij v_j with w the softmax of x over the keys that query i sees.  With
u = eps/2 of the type, for a kernel with f32 scores and sums:

* a score is off by dx <= D 2^-23 scale sum_d |q_d k_d| (f32 sums of D products) + 4 * 2^-23 max|x|
  (the steps after it, each relative to a value of at most max|x| or |scale q.k|) + 4e-7 softcap
  (tanh as 1 - 2 / (1 + e^2x) in f32); a weight then by 2 dx relative, its own and the sum's;
* exponentials are within 7.5e-5 (the polynomial of the tensor-core kernels) and weights
  are rounded to the type for the product: 7.5e-5 * 2 + u.  In f32 both are 3 * 2^-24;
* sums of n keys in f32: n 2^-23, and the store rounds by u |out|.

So |out - ref| <= u |ref| + (u_w + 2 (e + dx) + n 2^-23) sum_j w_ij |v_j|."""

import torch


def visible(B, Sq, Sk, causal=False, window=None, prefix=None, doc_ids=None, kv_lens=None, device="cuda"):
    lens = kv_lens.long().clamp(0, Sk) if kv_lens is not None else torch.full((B,), Sk, device=device)
    p = (lens[:, None] - Sq + torch.arange(Sq, device=device))[:, :, None]
    j = torch.arange(Sk, device=device)[None, None, :]
    near = torch.ones(B, Sq, Sk, dtype=torch.bool, device=device)
    if causal:
        near &= j <= p
    if window is not None:
        near &= (p - j).abs() < window
    if prefix is not None:
        pre = prefix.long()[:, None, None] if isinstance(prefix, torch.Tensor) else prefix
        near |= j < pre
    near &= j < lens[:, None, None]
    if doc_ids is not None:
        row = torch.gather(doc_ids.long(), 1, p[:, :, 0].clamp(0, max(Sk - 1, 0)))[:, :, None]
        near &= (p >= 0) & (row == doc_ids.long()[:, None, :]) & (row >= 0)
    return near, p, j


def reference(q, k, v, scale, softcap=None, slopes=None, **mask):
    """(out, bound) in 64 bits."""
    B, H, Sq, D = q.shape
    Hk, Sk = k.shape[1], k.shape[2]
    G = H // Hk
    near, p, j = visible(B, Sq, Sk, device=q.device, **mask)
    # what no query sees may hold anything
    used = near.any(1)[:, None, :, None]
    kd = torch.where(used, k.double(), 0.0).repeat_interleave(G, 1)
    vd = torch.where(used, v.double(), 0.0).repeat_interleave(G, 1)
    qd = q.double()
    raw = qd @ kd.transpose(-1, -2) * scale
    x = raw
    if softcap is not None:
        x = softcap * torch.tanh(x / softcap)
    if slopes is not None:
        x = x - slopes.double()[None, :, None, None] * (p - j).abs()[:, None].double()
    near = near[:, None]
    big = torch.where(near, torch.maximum(x.abs(), raw.abs()), 0.0).amax(-1, keepdim=True)
    terms = torch.where(near, (qd.abs() @ kd.abs().transpose(-1, -2)) * abs(scale), 0.0).amax(-1, keepdim=True)
    x = x.masked_fill(~near, float("-inf"))
    top = x.amax(-1, keepdim=True)
    w = torch.exp(x - torch.where(top == float("-inf"), 0.0, top))
    s = w.sum(-1, keepdim=True)
    w = w / torch.where(s == 0, 1.0, s)
    out, mag = w @ vd, w @ vd.abs()
    u = torch.finfo(q.dtype).eps / 2
    dx = D * 2.0 ** -23 * terms + 4 * 2.0 ** -23 * big + (4e-7 * softcap if softcap else 0.0)
    e, uw = (3 * 2.0 ** -24, 0.0) if q.dtype == torch.float32 else (7.5e-5, u)
    bound = u * 1.001 * out.abs() + (uw + 2 * (e + dx) + Sk * 2.0 ** -23) * mag
    fi = torch.finfo(q.dtype)
    return out, bound + fi.smallest_normal * fi.eps


def close(got, ref, bound):
    off = (got.double() - ref).abs()
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert (off <= bound).all(), f"off by {worst:.3g} times the bound"
