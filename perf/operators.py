"""What the operators of a quantised transformer block cost, and what they have to compute.

Three operators, used one after another in a block of a language model at inference:

* ``norm``: the residual's addition, a root-mean-square norm of the sum, and its output in the input's
  type or in 8 bits with one scale a token;
* ``linear``: the product of 8-bit activations (a scale a token) with 8-bit weights (a scale an output
  channel), rescaled and with the bias added;
* ``attention``: softmax attention with grouped heads over a sequence or a cache, whose scores may be
  capped by a tanh, get a bias that falls with the distance, and are masked (causal, window, prefix,
  document, cache lengths).

``listed`` are the cases that are measured, ``draw`` gives others of the same ranges, ``run`` makes one
pass: where ``own`` is false in elementary torch operations, where it is true through ``fusionpass_b200``.
"""

import math

import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"f16": 2, "bf16": 2, "f32": 4}


# ------------------------------------------------------------------ cases ---
def _norm(name, rows, cols, dtype, out, addends=2, total=True):
    return {"name": name, "op": "norm", "rows": rows, "cols": cols, "dtype": dtype, "out": out, "addends": addends,
            "sum": total}


def _linear(name, m, n, k, out, bias=False):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "out": out, "bias": bias}


def _attention(name, dtype, batch, heads, kv_heads, q_len, k_len, dim, cap=0.0, alibi=False, causal=False, window=0,
               prefix=0, docs=0, ragged=False):
    return {"name": name, "op": "attention", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "q_len": q_len, "k_len": k_len, "dim": dim, "cap": cap, "alibi": alibi, "causal": causal,
            "window": window, "prefix": prefix, "docs": docs, "ragged": ragged}


def listed():
    return [
        # one decoding step of 16 sequences: the residual and the branch, to 8 bits for the next product
        _norm("norm-decode-q8", 16, 4096, "f16", "q8"),
        # a batch of long prompts: what is read and written is all that counts
        _norm("norm-prompt-q8", 16384, 4096, "bf16", "q8"),
        # the last norm of a model: no residual kept, a width that no vector divides
        _norm("norm-odd", 1500, 2049, "f32", "y", addends=1, total=False),
        # one decoding step of 8 sequences: the weights are read once
        _linear("linear-decode", 8, 16384, 8192, "f16"),
        # a prompt of ordinary length
        _linear("linear-prompt", 1024, 4096, 4096, "bf16", bias=True),
        # the largest: a batch of long prompts through a wide layer
        _linear("linear-large", 8192, 8192, 8192, "f16"),
        # sizes that no tile divides, results kept in 32 bits
        _linear("linear-odd", 333, 1001, 1030, "f32", bias=True),
        # the first pass over a long prompt, grouped heads, capped scores
        _attention("attention-prompt-cap", "f16", 1, 32, 8, 8192, 8192, 128, cap=50.0, causal=True),
        # documents packed into rows for an encoder, scores that fall with the distance
        _attention("attention-documents", "bf16", 2, 16, 16, 4096, 4096, 64, alibi=True, docs=9),
        # a short prompt behind a cache, in a window, with a prefix that stays in sight, in 32 bits
        _attention("attention-prefix-odd", "f32", 2, 6, 3, 77, 130, 32, causal=True, window=30, prefix=41),
        # a piece of a prompt against a long cache, scores that fall with the distance
        _attention("attention-piece", "bf16", 1, 16, 4, 200, 32768, 128, alibi=True, causal=True),
        # one decoding step of 24 sequences of unequal length over their caches
        _attention("attention-decode-cap", "f16", 24, 32, 8, 1, 8192, 128, cap=30.0, causal=True, ragged=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "linear", "attention", "attention"])
    if op == "norm":
        dtype = rng.choice(["f16", "bf16", "f32"])
        cols = _log(rng, 64, 8192)
        rows = _log(rng, 1, min(20000, (1 << 26) // cols))
        out = "y" if dtype == "f32" else rng.choice(["y", "q8"])
        case = _norm("", rows, cols, dtype, out, rng.choice([1, 2, 2, 3]), rng.random() < 0.7)
    elif op == "linear":
        n, k = _log(rng, 64, 16384), _log(rng, 64, 8192)
        m = _log(rng, 1, min(8192, max(1, (1 << 38) // (n * k))))
        case = _linear("", m, n, k, rng.choice(["f16", "bf16", "f32"]), rng.random() < 0.5)
    else:
        dtype, dim = rng.choice(["f16", "bf16", "f32"]), rng.choice([16, 32, 64, 128])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 1, 2, 4, 8])
        top = (1 << 24) if dtype == "f32" else (1 << 28)
        k_len = _log(rng, 16, 32768)
        batch = rng.choice([1, 1, 2, 3, 8])
        most = max(1, min(k_len, top // (batch * heads * k_len)))
        q_len = 1 if rng.random() < 0.35 else _log(rng, 1, most)
        causal = rng.random() < 0.7
        case = _attention("", dtype, batch, heads, kv_heads, q_len, k_len, dim, cap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                          alibi=rng.random() < 0.4, causal=causal,
                          window=_log(rng, 1, k_len) if rng.random() < 0.3 else 0,
                          prefix=_log(rng, 1, k_len) if causal and rng.random() < 0.3 else 0,
                          docs=rng.randint(1, 12) if rng.random() < 0.3 else 0, ragged=rng.random() < 0.4)
    del case["name"]
    return case


# ----------------------------------------------------------------- inputs ---
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    if case["op"] == "norm":
        t = _TYPES[case["dtype"]]
        shape = (case["rows"], case["cols"])
        # a residual stream is several times as wide as a branch, and some channels stand out
        wide = 1.0 + 7.0 * (torch.rand(case["cols"], generator=g, device="cuda") > 0.995)
        addends = [(normal(*shape) * (3.0 * wide if i == 0 else 1.0)).to(t) for i in range(case["addends"])]
        return {"case": case, "addends": addends, "weight": (1.0 + 0.1 * normal(case["cols"])).to(t), "eps": 1e-6}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]

        def whole(rows):
            return normal(rows, k).mul_(40.0).round_().clamp_(-127, 127).to(torch.int8)

        x, w = whole(m), whole(n)
        xs = 0.02 + 0.02 * torch.rand(m, generator=g, device="cuda")
        ws = (0.5 + torch.rand(n, generator=g, device="cuda")) / (40.0 * math.sqrt(k))
        bias = normal(n).to(_TYPES[case["out"]]) if case["bias"] else None
        return {"case": case, "x": x, "x_scale": xs, "w": w, "w_scale": ws, "bias": bias}
    t = _TYPES[case["dtype"]]
    b, h, hk, sq, sk, d = (case[x] for x in ("batch", "heads", "kv_heads", "q_len", "k_len", "dim"))
    # with a cap, scores are as wide as the cap bites
    q = (normal(b, h, sq, d) * (8.0 if case["cap"] else 1.5)).to(t)
    k, v = normal(b, hk, sk, d).to(t), normal(b, hk, sk, d).to(t)
    lens = ids = slopes = None
    if case["ragged"]:
        # a sequence holds the new tokens at least, and three quarters of the cache on average
        low = max(sq, sk // 2)
        lens = torch.randint(low, sk + 1, (b,), generator=g, device="cuda").to(torch.int32)
    if case["docs"]:
        # documents of unequal length, one behind the other
        cuts = torch.rand(b, case["docs"] - 1, generator=g, device="cuda").mul_(sk).sort(dim=1).values
        at = torch.arange(sk, device="cuda", dtype=torch.float32).expand(b, sk).contiguous()
        ids = torch.searchsorted(cuts, at, right=True).to(torch.int32)
    if case["alibi"]:
        slopes = 2.0 ** (-8.0 * torch.arange(1, h + 1, device="cuda", dtype=torch.float32) / h)
    return {"case": case, "q": q, "k": k, "v": v, "scale": d ** -0.5, "lens": lens, "ids": ids, "slopes": slopes}


# -------------------------------------------------------------- one pass ---
def _of_8_bits(q, scale, dtype):
    """What 8-bit values with a scale a row stand for."""
    return torch.mul(q, scale.unsqueeze(-1), out=torch.empty(q.shape, dtype=dtype, device=q.device))


def _plain_norm(s):
    c = s["case"]
    t = _TYPES[c["dtype"]]
    total = s["addends"][0].float()
    if c["addends"] > 1:
        total = total + s["addends"][1].float()
    if c["addends"] > 2:
        total = total + s["addends"][2].float()
    y = total * torch.rsqrt(total.square().mean(-1, keepdim=True) + s["eps"]) * s["weight"].float()
    kept = [total.to(t)] if c["sum"] else []
    if c["out"] == "y":
        return [y.to(t)] + kept
    scale = y.abs().amax(-1) / 127.0
    q = torch.round(y / scale.unsqueeze(-1)).clamp(-127, 127)
    return [_of_8_bits(q, scale, t), scale] + kept


def _plain_linear(s):
    total = s["x"].float() @ s["w"].float().t()
    y = total * s["x_scale"].unsqueeze(-1) * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return [y.to(_TYPES[s["case"]["out"]])]


def _plain_attention(s):
    c = s["case"]
    b, h, hk, sq, sk, d = (c[x] for x in ("batch", "heads", "kv_heads", "q_len", "k_len", "dim"))
    g = h // hk
    scores = s["q"].float().reshape(b, hk, g * sq, d) @ s["k"].float().transpose(-1, -2)
    scores = (scores * s["scale"]).reshape(b, hk, g, sq, sk)
    if c["cap"]:
        scores = torch.tanh(scores / c["cap"]) * c["cap"]
    lens = s["lens"] if s["lens"] is not None else torch.full((b,), sk, device="cuda", dtype=torch.int32)
    at_q = lens[:, None] - sq + torch.arange(sq, device="cuda")
    at_k = torch.arange(sk, device="cuda")
    ahead = at_k - at_q[:, :, None]
    if s["slopes"] is not None:
        scores = scores - s["slopes"].reshape(1, hk, g, 1, 1) * ahead.abs()[:, None, None].float()
    seen = torch.ones_like(ahead, dtype=torch.bool)
    if c["causal"]:
        seen = seen & (ahead <= 0)
    if c["window"]:
        seen = seen & (ahead.abs() < c["window"])
    if c["prefix"]:
        seen = seen | (at_k < c["prefix"])
    seen = seen & (at_k < lens[:, None, None])
    if s["ids"] is not None:
        of_q = s["ids"].gather(1, at_q.clamp(min=0).long())
        seen = seen & (of_q[:, :, None] == s["ids"][:, None, :]) & (at_q[:, :, None] >= 0)
    scores = torch.where(seen[:, None, None], scores, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = p.reshape(b, hk, g * sq, sk) @ s["v"].float()
    out = out.reshape(b, h, sq, d) / torch.where(total == 0.0, 1.0, total).reshape(b, h, sq, 1)
    return [out.to(s["q"].dtype)]


def _own_norm(s):
    from fusionpass_b200 import fpkern

    c = s["case"]
    if c["out"] == "y":
        r = fpkern.add_rms_norm(s["addends"], s["weight"], s["eps"], return_sum=c["sum"])
        return list(r) if c["sum"] else [r]
    q, scale, *kept = fpkern.rms_norm_q8(s["addends"], s["weight"], s["eps"], return_sum=c["sum"])
    return [_of_8_bits(q, scale, _TYPES[c["dtype"]]), scale] + kept


def _own_linear(s):
    from fusionpass_b200 import fpkern

    return [fpkern.linear_q8(s["x"], s["x_scale"], s["w"], s["w_scale"], s["bias"],
                             out_dtype=_TYPES[s["case"]["out"]])]


def _own_attention(s):
    from fusionpass_b200 import fpkern

    c = s["case"]
    return [fpkern.score_attention(s["q"], s["k"], s["v"], s["scale"], softcap=c["cap"] or None, slopes=s["slopes"],
                                   causal=c["causal"], window=c["window"] or None, prefix=c["prefix"] or None,
                                   doc_ids=s["ids"], kv_lens=s["lens"])]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "linear": _own_linear, "attention": _own_attention}[op](state)
    return {"norm": _plain_norm, "linear": _plain_linear, "attention": _plain_attention}[op](state)


# ------------------------------------------------------------------- work ---
def _pairs(c):
    """Pairs of a query and a key that it sees, of one head of one sequence: with lengths and documents at
    their mean."""
    sq, sk = c["q_len"], c["k_len"]
    n = (max(sq, sk // 2) + sk) // 2 if c["ragged"] else sk
    at = torch.arange(sq, dtype=torch.float64) + (n - sq)
    high = at + 1 if c["causal"] else torch.full_like(at, n)
    low = torch.zeros_like(at)
    if c["window"]:
        high = torch.minimum(high, at + c["window"])
        low = (at - c["window"] + 1).clamp(min=0)
    high = high.clamp(max=n)
    seen = (high - low).clamp(min=0)
    if c["prefix"]:
        seen = seen + (torch.minimum(torch.tensor(float(min(c["prefix"], n))), low)
                       + (min(c["prefix"], n) - torch.maximum(high, low)).clamp(min=0))
    share = 1.0
    if c["docs"] > 1:
        # the mean over uniform cuts of the sum of squared lengths
        share = 2.0 / (c["docs"] + 1)
    return float(seen.sum()) * share, n


def work(case):
    if case["op"] == "norm":
        e, n = _SIZE[case["dtype"]], case["rows"] * case["cols"]
        written = n * e + (4 * case["rows"] if case["out"] == "q8" else 0) + (n * e if case["sum"] else 0)
        return {"bytes": case["addends"] * n * e + case["cols"] * e + written, "flops": (case["addends"] + 5) * n}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        e = _SIZE[case["out"]]
        return {"bytes": m * k + n * k + 4 * (m + n) + m * n * e + (n * e if case["bias"] else 0),
                "flops": 2 * m * n * k}
    e = _SIZE[case["dtype"]]
    pairs, n = _pairs(case)
    rows = case["batch"] * case["heads"] * case["q_len"] * case["dim"]
    kept = n
    if case["window"] and case["causal"]:
        kept = min(n, case["q_len"] + case["window"] - 1 + case["prefix"])
    caches = case["batch"] * case["kv_heads"] * kept * case["dim"]
    return {"bytes": 2 * rows * e + 2 * caches * e, "flops": 4 * case["batch"] * case["heads"] * pairs * case["dim"]}


# ------------------------------------------------------------ in 64 bits ---
def exact(case, seed):
    """The same from the definitions, in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "norm":
        x = s["addends"][0].double()
        for t in s["addends"][1:]:
            x += t
        y = s["weight"].double() * x / ((x * x).sum(-1, keepdim=True) / case["cols"] + s["eps"]).sqrt()
        if case["out"] == "y":
            outs = [y]
        else:
            step = y.abs().max(-1, keepdim=True).values / 127
            outs = [(y / step).round() * step, step.squeeze(-1)]
        return outs + ([x] if case["sum"] else [])
    if case["op"] == "linear":
        y = torch.einsum("mk,nk->mn", s["x"].double(), s["w"].double())
        y = y * torch.outer(s["x_scale"].double(), s["w_scale"].double())
        return [y if s["bias"] is None else y + s["bias"].double()]
    b, h, hk, sq, sk, d = (case[x] for x in ("batch", "heads", "kv_heads", "q_len", "k_len", "dim"))
    out = torch.zeros(b, h, sq, d, device="cuda", dtype=torch.float64)
    for i in range(b):
        n = int(s["lens"][i]) if s["lens"] is not None else sk
        row = torch.arange(n - sq, n, device="cuda")[:, None]
        col = torch.arange(n, device="cuda")[None, :]
        near = torch.ones(sq, n, device="cuda", dtype=torch.bool)
        if case["causal"]:
            near &= col <= row
        if case["window"]:
            near &= ((row - col) < case["window"]) & ((col - row) < case["window"])
        if case["prefix"]:
            near |= col < case["prefix"]
        if s["ids"] is not None:
            ids = s["ids"][i, :n]
            near &= ids[n - sq:, None] == ids[None, :]
        for j in range(h):
            z = (s["q"][i, j].double() @ s["k"][i, j * hk // h, :n].double().t()) * s["scale"]
            if case["cap"]:
                z = case["cap"] * torch.tanh(z / case["cap"])
            if s["slopes"] is not None:
                z = z - s["slopes"][j].double() * (row - col).abs()
            z = z.masked_fill(~near, float("-inf"))
            # a row that sees nothing gives zeros
            w = torch.softmax(z, -1).nan_to_num(nan=0.0)
            out[i, j] = w @ s["v"][i, j * hk // h, :n].double()
    return [out]
