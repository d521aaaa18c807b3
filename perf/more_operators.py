"""What the operators of speculative decoding over an 8-bit cache cost, and what they have to compute.

Five operators, used one after another in a decoding step that drafts a tree of tokens:

* ``cache``: new keys and values quantised as they are written into a cache (8 bits, a scale a row), the rows of
  the accepted branch moved up behind the rows that were there, and the cache read back in the model's type, as
  attention over a prompt that is taken in pieces needs it;
* ``tree``: attention of a tree of drafted tokens over a cache, in 8 bits or in the model's type: a node sees what
  was there before, its ancestors and itself; a tree of one node is an ordinary decoding step;
* ``verify``: which drafted tokens the target's probabilities accept, from given random numbers, and the next token.

``listed`` are the cases that are measured, ``draw`` gives others of the same ranges, ``run`` makes one pass:
where ``own`` is false in elementary torch operations, where it is true through ``fusionpass_b200``.
"""

import math

import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"f16": 2, "bf16": 2, "f32": 4}


# ------------------------------------------------------------------ cases ---
def _cache(name, dtype, batch, kv_heads, room, new, dim, keep=False, ragged=False):
    return {"name": name, "op": "cache", "dtype": dtype, "batch": batch, "kv_heads": kv_heads, "room": room,
            "new": new, "dim": dim, "keep": keep, "ragged": ragged}


def _tree(name, dtype, batch, heads, kv_heads, nodes, room, dim, q8=True, ragged=False):
    return {"name": name, "op": "tree", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "nodes": nodes, "room": room, "dim": dim, "q8": q8, "ragged": ragged}


def _verify(name, batch, nodes, vocab, draft=True):
    return {"name": name, "op": "verify", "batch": batch, "nodes": nodes, "vocab": vocab, "draft": draft}


def listed():
    return [
        # a batch of long prompts written whole: what is read and written is all that counts
        _cache("cache-prompt", "f16", 2, 8, 8192, 8192, 128),
        # one step of 16 sequences: their drafted tokens, the branches that were accepted
        _cache("cache-step", "bf16", 16, 8, 2048, 16, 128, keep=True, ragged=True),
        # odd sizes in 32 bits, where latency counts
        _cache("cache-odd", "f32", 3, 2, 333, 21, 64, keep=True, ragged=True),
        # single tokens: a decoding step of 24 sequences of unequal length
        _tree("tree-token", "f16", 24, 32, 8, 1, 8192, 128, ragged=True),
        # a small tree of one sequence over a short cache in the model's type, where latency counts
        _tree("tree-small", "bf16", 1, 32, 8, 8, 2048, 128, q8=False),
        # an ordinary step
        _tree("tree-step", "f16", 16, 32, 8, 16, 4096, 128, ragged=True),
        # small heads, a cache in the model's type, a tree that fills no tile
        _tree("tree-16bit", "bf16", 8, 32, 8, 49, 8192, 64, q8=False, ragged=True),
        # the largest: wide trees over long caches
        _tree("tree-large", "f16", 8, 32, 8, 64, 16384, 128),
        # odd sizes, all in 32 bits but the cache
        _tree("tree-odd", "f32", 2, 6, 3, 21, 333, 32, ragged=True),
        # one sequence, a small tree, where latency counts
        _verify("verify-one", 1, 8, 32000),
        # a batch with a large vocabulary
        _verify("verify-batch", 32, 32, 131072),
        # tokens that were drafted without probabilities, a vocabulary of odd size
        _verify("verify-certain", 16, 24, 50001, draft=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["cache", "tree", "tree", "verify"])
    if op == "cache":
        dtype, dim = rng.choice(["f16", "bf16", "f32"]), rng.choice([16, 32, 64, 128])
        kv_heads, batch = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 8, 16])
        room = _log(rng, 16, min(32768, (1 << 24) // (kv_heads * batch * dim)))
        new = room if rng.random() < 0.3 else _log(rng, 1, room)
        case = _cache("", dtype, batch, kv_heads, room, new, dim, keep=new <= 256 and rng.random() < 0.6,
                      ragged=rng.random() < 0.5)
    elif op == "tree":
        dtype, dim = rng.choice(["f16", "bf16", "f32"]), rng.choice([16, 32, 64, 128])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 1, 2, 4, 8])
        batch = rng.choice([1, 1, 2, 3, 8, 24])
        room = _log(rng, 16, 32768)
        top = (1 << 24) if dtype == "f32" else (1 << 27)
        most = max(1, min(256, room, top // (batch * heads * room)))
        nodes = 1 if rng.random() < 0.25 else _log(rng, 1, most)
        case = _tree("", dtype, batch, heads, kv_heads, nodes, room, dim, q8=rng.random() < 0.6,
                     ragged=rng.random() < 0.5)
    else:
        batch, vocab = rng.choice([1, 1, 2, 5, 16, 32]), _log(rng, 100, 131072)
        case = _verify("", batch, _log(rng, 1, max(1, min(64, (1 << 26) // (batch * vocab)))), vocab,
                       draft=rng.random() < 0.6)
    del case["name"]
    return case


# ----------------------------------------------------------------- inputs ---
def _quantised(x):
    """int8 rows and a scale a row of what a cache holds already."""
    top = x.abs().amax(-1)
    return torch.round(x * (127.0 / top).unsqueeze(-1)).clamp_(-127, 127).to(torch.int8), top / 127.0


def _parents(batch, nodes, g):
    """Trees: node 0 is the root, and a later node hangs on an earlier one, more often on a late one."""
    i = torch.arange(nodes, device="cuda")
    at = (i * torch.rand(batch, nodes, generator=g, device="cuda").sqrt()).long().minimum((i - 1).clamp(min=0))
    at[:, 0] = -1
    return at.to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def whole(low, high, *shape):
        return torch.randint(low, high + 1, shape, generator=g, device="cuda").to(torch.int32)

    b = case["batch"]
    if case["op"] == "verify":
        t, v = case["nodes"], case["vocab"]
        # the draft follows the target, not exactly; both are as peaked as a language model's
        logits = 3.0 * normal(b, t, v)
        target = torch.softmax(logits, -1)
        draft = torch.softmax(logits + 0.7 * normal(b, t, v), -1)
        parents = _parents(b, t, g)
        drawn = torch.multinomial(draft.reshape(b * t, v), 4, replacement=True, generator=g).reshape(b, t, 4)
        of = parents.long().clamp(min=0)
        which = (torch.arange(t, device="cuda") % 4).expand(b, t)
        tokens = drawn.gather(1, of.unsqueeze(-1).expand(b, t, 4)).gather(2, which.unsqueeze(-1)).squeeze(-1)
        lens = whole(max(1, t // 2), t, b)
        return {"case": case, "tokens": tokens.to(torch.int32), "parents": parents, "target": target,
                "draft": draft if case["draft"] else None, "lens": lens,
                "uniform": torch.rand(b, t, generator=g, device="cuda")}
    t, hk, n, d = _TYPES[case["dtype"]], case["kv_heads"], case["room"], case["dim"]
    new = case["new"] if case["op"] == "cache" else case["nodes"]
    past = torch.full((b,), n - new, dtype=torch.int32, device="cuda")
    lens = torch.full((b,), new, dtype=torch.int32, device="cuda")
    if case["ragged"]:
        # at least half of the room was filled; a sequence has fewer new rows than there is place for
        past = whole((n - new) // 2, n - new, b)
        lens = whole((new + 1) // 2, new, b)
    # keys have channels that stand out, values do not
    wide = 1.0 + 4.0 * (torch.rand(hk, 1, d, generator=g, device="cuda") > 0.97)
    keys, values = normal(b, hk, n, d) * wide, normal(b, hk, n, d)
    if case["op"] == "cache":
        (kc, ks), (vc, vs) = _quantised(keys), _quantised(values)
        # a branch of the tree: rows in rising order, the first of them first
        steps = whole(1, 3, b, new)
        path = steps.cumsum(1) - steps[:, :1]
        path = torch.where(path < lens.unsqueeze(1), path, -1).to(torch.int32)
        counts = torch.minimum(whole(1, new // 2 + 1, b), (path >= 0).sum(1)).to(torch.int32)
        return {"case": case, "k": (normal(b, hk, new, d) * wide).to(t), "v": normal(b, hk, new, d).to(t), "past": past,
                "lens": lens, "path": path, "counts": counts, "k_cache": kc, "v_cache": vc, "k_scale": ks, "v_scale": vs,
                "kv_lens": past + (counts if case["keep"] else lens)}
    ks = vs = None
    if case["q8"]:
        (k, ks), (v, vs) = _quantised(keys), _quantised(values)
    else:
        k, v = keys.to(t), values.to(t)
    return {"case": case, "q": (1.5 * normal(b, case["heads"], new, d)).to(t), "k": k, "v": v, "k_scale": ks,
            "v_scale": vs, "scale": d ** -0.5, "parents": _parents(b, new, g), "past": past, "lens": lens}


# -------------------------------------------------------------- one pass ---
def _write(x, cache, scale, at, fresh):
    """Rows ``x`` in 8 bits to rows ``at`` of the cache where ``fresh``."""
    x = x.double()  # a value next to the middle of two whole numbers goes to the right one
    top = x.abs().amax(-1, keepdim=True)
    q = torch.round(x * 127.0 / torch.where(top > 0.0, top, 1.0)).to(torch.int8)
    one = (top / 127.0).float().squeeze(-1)
    rows = at.unsqueeze(-1).expand_as(q)
    cache.scatter_(2, rows, torch.where(fresh.unsqueeze(-1), q, cache.gather(2, rows)))
    scale.scatter_(2, at, torch.where(fresh, one, scale.gather(2, at)))


def _move(cache, source, at, kept):
    """Row ``source`` to row ``at`` where ``kept``."""
    if cache.dim() == 4:
        source, at, kept = (x.unsqueeze(-1).expand(*x.shape, cache.shape[-1]) for x in (source, at, kept))
    cache.scatter_(2, at, torch.where(kept, cache.gather(2, source), cache.gather(2, at)))


def _plain_cache(s):
    c = s["case"]
    b, hk, n, new, t = c["batch"], c["kv_heads"], c["room"], c["new"], _TYPES[c["dtype"]]
    i = torch.arange(new, device="cuda")
    at = (s["past"].long()[:, None] + i)[:, None].expand(b, hk, new)
    fresh = (i < s["lens"][:, None])[:, None].expand(b, hk, new)
    _write(s["k"], s["k_cache"], s["k_scale"], at, fresh)
    _write(s["v"], s["v_cache"], s["v_scale"], at, fresh)
    if c["keep"]:
        kept = (i < s["counts"][:, None])[:, None].expand(b, hk, new)
        source = (s["past"][:, None] + s["path"].clamp(min=0)).long()[:, None].expand(b, hk, new)
        _move(s["k_cache"], source, at, kept)
        _move(s["v_cache"], source, at, kept)
        _move(s["k_scale"], source, at, kept)
        _move(s["v_scale"], source, at, kept)
    held = (torch.arange(n, device="cuda") < s["kv_lens"][:, None])[:, None, :, None]
    k = torch.where(held, s["k_cache"].float() * s["k_scale"].unsqueeze(-1), 0.0).to(t)
    v = torch.where(held, s["v_cache"].float() * s["v_scale"].unsqueeze(-1), 0.0).to(t)
    return [k, v, s["k_scale"], s["v_scale"]]


def _ancestors(parents):
    """[B, T, T]: node j is node i or one of its ancestors."""
    b, t = parents.shape
    i = torch.arange(t, device=parents.device)
    m = ((parents.long()[:, :, None] == i) | (i[:, None] == i)).float()
    for _ in range(max(1, (t - 1).bit_length())):  # paths of up to 1, 2, 4, ... edges
        m = ((m @ m) > 0.0).float()
    return m > 0.0


def _plain_tree(s):
    c = s["case"]
    b, h, hk, t, n, d = (c[x] for x in ("batch", "heads", "kv_heads", "nodes", "room", "dim"))
    k, v = s["k"].float(), s["v"].float()
    if c["q8"]:
        k, v = k * s["k_scale"].unsqueeze(-1), v * s["v_scale"].unsqueeze(-1)
    node = torch.arange(n, device="cuda") - s["past"][:, None]  # what node of its tree a row is
    real = (node >= 0) & (node < s["lens"][:, None])
    up = _ancestors(s["parents"]).gather(2, node.clamp(0, t - 1)[:, None].expand(b, t, n))
    seen = (node < 0)[:, None] | (real[:, None] & up)
    seen = seen & (torch.arange(t, device="cuda") < s["lens"][:, None])[:, :, None]
    scores = s["q"].float().reshape(b, hk, h // hk * t, d) @ k.transpose(-1, -2)
    scores = (scores * s["scale"]).reshape(b, hk, h // hk, t, n)
    scores = torch.where(seen[:, None, None], scores, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = (p.reshape(b, hk, h // hk * t, n) @ v).reshape(b, h, t, d)
    return [(out / torch.where(total == 0.0, 1.0, total).reshape(b, h, t, 1)).to(s["q"].dtype)]


def _plain_verify(s):
    c = s["case"]
    b, t = c["batch"], c["nodes"]
    rows = torch.arange(b, device="cuda")
    tokens, parents, lens = s["tokens"].long(), s["parents"].long(), s["lens"].long()
    u = s["uniform"].double()
    at = torch.zeros(b, dtype=torch.long, device="cuda")
    path = torch.full((b, t), -1, dtype=torch.long, device="cuda")
    path[:, 0] = 0
    counts = torch.ones(b, dtype=torch.long, device="cuda")
    left = s["target"][:, 0].double()  # of the target's probabilities, where the drafts that failed are taken out
    mass = torch.ones(b, dtype=torch.float64, device="cuda")
    for i in range(1, t):  # a node comes after its parent and its earlier siblings
        child = (parents[:, i] == at) & (i < lens)
        token = tokens[:, i]
        if s["draft"] is not None:
            q = s["draft"][rows, at].double()
        else:
            q = torch.zeros_like(left).scatter_(1, token[:, None], 1.0)
        r = left[rows, token]
        taken = child & (u[:, i] * q[rows, token] * mass < r)
        failed = child & ~taken
        rest = torch.where(failed[:, None], (left - mass[:, None] * q).clamp(min=0.0), left)
        mass = torch.where(failed, rest.sum(-1), mass)
        at = torch.where(taken, i, at)
        left = torch.where(taken[:, None], s["target"][:, i].double(), rest)
        mass = torch.where(taken, 1.0, mass)
        path.scatter_(1, counts.clamp(max=t - 1)[:, None], torch.where(taken, i, path[rows, counts.clamp(max=t - 1)])[:, None])
        counts = counts + taken
    cdf = left.cumsum(-1)
    token = (cdf <= u[:, :1] * cdf[:, -1:]).sum(-1)
    return [path.to(torch.int32), counts.to(torch.int32), token.to(torch.int32)]


def _own_cache(s):
    from fusionpass_b200 import fpkern

    caches = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    fpkern.cache_write_q8(s["k"], s["v"], *caches, s["past"], new_lens=s["lens"])
    if s["case"]["keep"]:
        fpkern.cache_keep(caches, s["path"], s["counts"], s["past"])
    k, v = fpkern.cache_read_q8(*caches, dtype=_TYPES[s["case"]["dtype"]], kv_lens=s["kv_lens"])
    return [k, v, s["k_scale"], s["v_scale"]]


def _own_tree(s):
    from fusionpass_b200 import fpkern

    return [fpkern.tree_attention(s["q"], s["k"], s["v"], s["scale"], s["parents"], s["past"], tree_lens=s["lens"],
                                  k_scale=s["k_scale"], v_scale=s["v_scale"])]


def _own_verify(s):
    from fusionpass_b200 import fpkern

    return list(fpkern.verify_draft(s["tokens"], s["parents"], s["target"], s["draft"], s["uniform"],
                                    tree_lens=s["lens"]))


def run(state):
    op = state["case"]["op"]
    if own:
        return {"cache": _own_cache, "tree": _own_tree, "verify": _own_verify}[op](state)
    return {"cache": _plain_cache, "tree": _plain_tree, "verify": _plain_verify}[op](state)


# ------------------------------------------------------------------- work ---
def work(case):
    if case["op"] == "verify":
        b, t, v = case["batch"], case["nodes"], case["vocab"]
        # the row that the last token is drawn from, of both where drafts failed there; the rest are gathers
        rows = 2 if case["draft"] else 1
        return {"bytes": b * (4 * v * rows + 8 * 3 * t), "flops": 4 * b * v}
    e, b, hk, n, d = _SIZE[case["dtype"]], case["batch"], case["kv_heads"], case["room"], case["dim"]
    new = case["new"] if case["op"] == "cache" else case["nodes"]
    past = n - new
    if case["ragged"]:  # at their mean
        past, new = past * 3 // 4, max(1, new * 3 // 4)
    if case["op"] == "cache":
        # new rows read and written; what was there read; the room's rows written in the model's type
        moved = 2 * b * hk * (new * (d * e + d + 4) + past * (d + 4) + n * d * e)
        return {"bytes": moved, "flops": 2 * b * hk * d * (4 * new + past + new)}
    row = d + 4 if case["q8"] else d * e
    h = case["heads"]
    pairs = new * past + new * (new + 1) // 2
    return {"bytes": 2 * b * h * new * d * e + 2 * b * hk * (past + new) * row, "flops": 4 * b * h * pairs * d}


# ------------------------------------------------------------ in 64 bits ---
def _exact_cache(case, s):
    values, scales = [], []
    for new, q, scale in ((s["k"], s["k_cache"], s["k_scale"]), (s["v"], s["v_cache"], s["v_scale"])):
        whole, step = q.double(), scale.double()
        for b in range(case["batch"]):
            n, m = int(s["past"][b]), int(s["lens"][b])
            x = new[b, :, :m].double()
            one = x.abs().max(-1).values / 127
            whole[b, :, n:n + m] = (x / one.unsqueeze(-1)).round()
            step[b, :, n:n + m] = one
            if case["keep"]:
                source = n + s["path"][b, :int(s["counts"][b])].long()
                whole[b, :, n:n + len(source)] = whole[b, :, source]
                step[b, :, n:n + len(source)] = step[b, :, source]
        value = whole * step.unsqueeze(-1)
        for b in range(case["batch"]):
            value[b, :, int(s["kv_lens"][b]):] = 0
        values.append(value)
        scales.append(step)
    return values + scales


def _exact_tree(case, s):
    b, h, t, d = (case[x] for x in ("batch", "heads", "nodes", "dim"))
    out = torch.zeros(b, h, t, d, device="cuda", dtype=torch.float64)
    for i in range(b):
        n, m = int(s["past"][i]), int(s["lens"][i])
        up = s["parents"][i].tolist()
        near = torch.zeros(m, n + m, dtype=torch.bool)
        near[:, :n] = True
        for x in range(m):
            y = x
            while y >= 0:
                near[x, n + y] = True
                y = up[y]
        near = near.cuda()
        for j in range(h):
            kv = j * case["kv_heads"] // h
            k, v = s["k"][i, kv, :n + m].double(), s["v"][i, kv, :n + m].double()
            if case["q8"]:
                k, v = k * s["k_scale"][i, kv, :n + m, None].double(), v * s["v_scale"][i, kv, :n + m, None].double()
            z = (s["q"][i, j, :m].double() @ k.t()) * s["scale"]
            out[i, j, :m] = torch.softmax(z.masked_fill(~near, float("-inf")), -1) @ v
    return [out]


def _exact_verify(case, s):
    paths, counts, last = [], [], []
    for b in range(case["batch"]):
        parents, tokens, u = s["parents"][b].tolist(), s["tokens"][b].tolist(), s["uniform"][b].double().tolist()
        path, seeking = [0], True
        while seeking:
            seeking = False
            here = path[-1]
            p, m = s["target"][b, here].double(), 1.0
            for x in [y for y in range(here + 1, int(s["lens"][b])) if parents[y] == here]:
                if s["draft"] is not None:
                    q = s["draft"][b, here].double()
                else:
                    q = torch.nn.functional.one_hot(torch.tensor(tokens[x], device="cuda"), case["vocab"]).double()
                if u[x] * float(q[tokens[x]]) * m < float(p[tokens[x]]):
                    path.append(x)
                    seeking = True
                    break
                p = (p - m * q).clamp(min=0)
                m = float(p.sum())
        cdf = torch.cumsum(p, 0)
        last.append(int(torch.searchsorted(cdf, (cdf[-1] * u[0]).reshape(1), right=True)))
        paths.append(path + [-1] * (case["nodes"] - len(path)))
        counts.append(len(path))
    return [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (paths, counts, last)]


def exact(case, seed):
    """The same from the definitions, in 64 bits."""
    s = prepare(case, seed)
    return {"cache": _exact_cache, "tree": _exact_tree, "verify": _exact_verify}[case["op"]](case, s)
