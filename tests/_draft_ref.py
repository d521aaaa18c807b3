"""The 8-bit cache, tree attention and the verification of drafted tokens from their definitions in
64 bits, and the bound of a tree attention kernel's error.

out_i = sum_j w_ij v_j with w the softmax of x = scale q.k over the keys that node i sees, k and v
q8 * scale for an 8-bit cache.  With u = eps/2 of the type, for a kernel with f32 scores and sums:

* a score is off by dx <= D 2^-23 sum_d |scale q_d k_d| (f32 sums of D products, an ulp each, and
  the scale's product) + 4 * 2^-23 max|x| (its factors, the difference to the maximum, the
  maximum's change of base, each a rounding of a value of at most max|x|, or twice that);
* exponentials are within 2^-22 (ex2.approx, expf), and so are the factors with which parts are
  joined or scaled anew, of which a key meets at most three that its neighbours do not (a new
  maximum, its warp's or part's, the last joining): e = 4 * 2^-22.  A weight is off by
  2 (e + dx), its own and the sum's;
* for the product with v weights are rounded to the type, u, after at most three f32 products with
  the value's scale (3 * 2^-24); in f32 v itself is rounded once (2^-24).  In f16 weights are held
  below 2^-14 in steps of 2^-24, half of one each; with 8 bits they stand for parts of a power of two
  of at most twice the largest scale: 2 * 2^-25 max|v| a key, while the largest weight, and so their
  sum, is at least 1;
* sums of n keys in f32: n 2^-23; the store rounds by u |out|, the division by 2^-23 |out|."""

import torch


def quantised(x):
    """(q, scale) of the rows of x: 127 x / top is right to 2^-52 in 64 bits, and two whole numbers'
    middle is at least 2^-33 away from any other such quotient of 24-bit numbers."""
    d = x.double()
    top = d.abs().amax(-1)
    odd, none = ~torch.isfinite(top), top < 127 * torch.finfo(torch.float32).smallest_normal
    q = torch.round(d * 127.0 / torch.where(odd | none, 1.0, top).unsqueeze(-1))
    q = torch.where((odd | none).unsqueeze(-1), 0.0, q).to(torch.int8)
    scale = torch.where(odd, float("nan"), torch.where(none, 0.0, top / 127.0)).float()
    return q, scale


def sight(parents, past, lens, room):
    """[B, T, room] truth values: node i sees row j."""
    B, T = parents.shape
    near = torch.zeros(B, T, room, dtype=torch.bool)
    for b in range(B):
        n, p = min(max(int(lens[b]), 0), T), int(past[b])
        for i in range(n):
            near[b, i, :max(min(p, room), 0)] = True
            a = i
            while True:
                if 0 <= p + a < room:
                    near[b, i, p + a] = True
                up = int(parents[b, a])
                if not 0 <= up < a:
                    break
                a = up
    return near


def tree_reference(q, k, v, scale, near, k_scale=None, v_scale=None):
    """(out, bound) in 64 bits; what no node sees may hold anything."""
    B, H, T, D = q.shape
    Hk, N = k.shape[1], k.shape[2]
    near = near.to(q.device)
    used = near.any(1)[:, None, :, None]
    kd, vd = k.double(), v.double()
    if k_scale is not None:
        kd, vd = kd * k_scale.double().unsqueeze(-1), vd * v_scale.double().unsqueeze(-1)
    kd, vd = (torch.where(used, t, 0.0).repeat_interleave(H // Hk, 1) for t in (kd, vd))
    qd, near = q.double(), near[:, None]
    x = qd @ kd.transpose(-1, -2) * scale
    big = torch.where(near, x.abs(), 0.0).amax(-1, keepdim=True)
    terms = torch.where(near, (qd.abs() @ kd.abs().transpose(-1, -2)) * abs(scale), 0.0).amax(-1, keepdim=True)
    x = x.masked_fill(~near, float("-inf"))
    top = x.amax(-1, keepdim=True)
    w = torch.exp(x - torch.where(top == float("-inf"), 0.0, top))
    s = w.sum(-1, keepdim=True)
    w = w / torch.where(s == 0, 1.0, s)
    out, mag = w @ vd, w @ vd.abs()
    u = torch.finfo(q.dtype).eps / 2
    dx = D * 2.0 ** -23 * terms + 4 * 2.0 ** -23 * big
    bound = (u + 2.0 ** -23) * out.abs() + (u + 3 * 2.0 ** -24 + 2 * (4 * 2.0 ** -22 + dx) + N * 2.0 ** -23) * mag
    if q.dtype == torch.float16:
        seen = near.any(-1, keepdim=True)
        bound = bound + torch.where(seen, N * 2.0 ** -24, 0.0) * vd.abs().amax((2, 3), keepdim=True)
    fi = torch.finfo(q.dtype)
    return out, bound * (1 + 2 * u) + fi.smallest_normal * fi.eps


def verify_reference(tokens, parents, target, draft, uniform, lens):
    """(path, counts, next) of one sequence after the other, r made anew step by step."""
    B, T, V = target.shape
    paths, counts, nexts = [], [], []
    for b in range(B):
        n = min(max(int(lens[b]), 0), T)
        if n == 0:
            paths.append([-1] * T)
            counts.append(0)
            nexts.append(-1)
            continue
        path = [0]
        walking = True
        while walking:
            walking = False
            at = path[-1]
            r, m = target[b, at].double().nan_to_num(0.0, float("inf")).clamp(min=0), 1.0
            for x in range(at + 1, n):
                tok = int(tokens[b, x])
                if int(parents[b, x]) != at or not 0 <= tok < V:
                    continue
                if draft is not None:
                    q = draft[b, at].double().nan_to_num(0.0, float("inf")).clamp(min=0)
                else:
                    q = torch.zeros(V, dtype=torch.float64, device=target.device)
                    q[tok] = 1.0
                if float(uniform[b, x].double()) * float(q[tok]) * m < float(r[tok]):
                    path.append(x)
                    walking = True
                    break
                r = (r - m * q).clamp(min=0)
                m = float(r.sum())
            if not walking:
                break
        total = float(r.sum())
        nxt = -1
        if 0.0 < total < float("inf"):
            u = min(max(0.0, float(uniform[b, 0])), 1.0 - 2.0 ** -24)  # NaN: 0
            run = r.cumsum(0)
            nxt = int((run <= u * float(run[-1])).sum())
        paths.append(path + [-1] * (T - len(path)))
        counts.append(len(path))
        nexts.append(nxt)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return i32(paths).reshape(B, T), i32(counts), i32(nexts)


def close(got, ref, bound):
    off = (got.double() - ref).abs()
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert (off <= bound).all(), f"off by {worst:.3g} times the bound"
