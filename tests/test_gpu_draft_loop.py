"""GPU: the operators of speculative decoding used one after another, as a program uses them: eagerly,
captured and replayed, on other streams."""

import pytest
import torch

from fusionpass_b200 import fpkern
from tests._draft_ref import close, quantised, sight, tree_reference, verify_reference

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
TREE = [-1, 0, 0, 1, 1, 2, 3, 5]


class Toy:
    """A model of one attention layer: a token's key, value and query are rows of tables, and its
    probabilities a softmax over what its queries' heads saw."""

    def __init__(self, dt, V, H, Hk, D, g):
        r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
        self.q, self.k, self.v = r(V, H, D).to(dt), r(V, Hk, D).to(dt), r(V, Hk, D).to(dt)
        self.head = r(H * D, V) * 0.5
        self.scale = D ** -0.5

    def rows(self, tokens):
        pick = lambda t: t[tokens.long()].transpose(1, 2)  # noqa: E731
        return pick(self.q), pick(self.k), pick(self.v)

    def probabilities(self, out):
        b, h, t, d = out.shape
        return torch.softmax(out.transpose(1, 2).reshape(b, t, h * d).float() @ self.head, -1)


def step(toy, caches, tokens, parents, past, uniform, draft):
    q, k, v = toy.rows(tokens)
    fpkern.cache_write_q8(k, v, *caches, past)
    out = fpkern.tree_attention(q, caches[0], caches[1], toy.scale, parents, past, k_scale=caches[2], v_scale=caches[3])
    path, counts, nxt = fpkern.verify_draft(tokens, parents, toy.probabilities(out), draft, uniform)
    fpkern.cache_keep(caches, path, counts, past)
    return out, path, counts, nxt


def _state(dt, B, V, H, Hk, D, N, g):
    toy = Toy(dt, V, H, Hk, D, g)
    caches = tuple(torch.zeros(B, Hk, N, D, dtype=torch.int8, device="cuda") for _ in range(2)) + \
        tuple(torch.zeros(B, Hk, N, device="cuda") for _ in range(2))
    return toy, caches


@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("heads", [(4, 2), (16, 2)])
@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_generation(dt, heads, with_draft):
    """Several steps: at each the cache's rows are those of the accepted tokens, each node's result is that of
    its own path, and the walk that of the probabilities."""
    B, V, D, N, T = 3, 64, 64, 200, len(TREE)
    g = torch.Generator(device="cuda").manual_seed(heads[0] + with_draft)
    toy, caches = _state(dt, B, V, *heads, D, N, g)
    rnd = lambda *s: torch.randint(0, V, s, generator=g, device="cuda").to(torch.int32)  # noqa: E731
    prompt = rnd(B, 40)
    _, k, v = toy.rows(prompt)
    past = torch.tensor([40, 17, 1], dtype=torch.int32, device="cuda")
    fpkern.cache_write_q8(k, v, *caches, torch.zeros(B, dtype=torch.int32, device="cuda"), new_lens=past)
    said = [prompt[b, :past[b]].tolist() for b in range(B)]
    last = rnd(B)
    parents = torch.tensor(TREE, dtype=torch.int32, device="cuda")
    for _ in range(4):
        tokens = rnd(B, T)
        tokens[:, 0] = last
        uniform = torch.rand(B, T, generator=g, device="cuda") * 0.3
        draft = torch.softmax(torch.randn(B, T, V, generator=g, device="cuda"), -1) if with_draft else None
        out, path, counts, nxt = step(toy, caches, tokens, parents, past, uniform, draft)
        # the tree's attention, from the tokens alone
        seqs = [torch.tensor(said[b] + tokens[b].tolist(), device="cuda") for b in range(B)]
        full = torch.zeros(B, max(len(s) for s in seqs), dtype=torch.int64, device="cuda")
        for b, s in enumerate(seqs):
            full[b, :len(s)] = s
        q, _, _ = toy.rows(tokens)
        _, k, v = toy.rows(full)
        (k8, ks), (v8, vs) = quantised(k), quantised(v)
        near = sight(parents.expand(B, T), past, [T] * B, full.shape[1])
        ref, bound = tree_reference(q, k8, v8, toy.scale, near, ks, vs)
        close(out, ref, bound)
        want = verify_reference(tokens, parents.expand(B, T), toy.probabilities(out), draft, uniform, [T] * B)
        for a, b in zip((path, counts, nxt), want):
            assert torch.equal(a.cpu(), b)
        for b in range(B):
            said[b] += tokens[b, path[b, :counts[b]].long()].tolist()
        past = past + counts
        last = nxt
        for b in range(B):
            assert past[b] == len(said[b])
            _, k, v = toy.rows(torch.tensor([said[b]], device="cuda"))
            for x, c, s in ((k, caches[0], caches[2]), (v, caches[1], caches[3])):
                w8, w1 = quantised(x)
                assert torch.equal(c[b, :, :len(said[b])], w8[0]) and torch.equal(s[b, :, :len(said[b])], w1[0])
    k, v = fpkern.cache_read_q8(*caches, dtype=dt, kv_lens=past)
    assert torch.equal(k, torch.where(torch.arange(N, device="cuda")[:, None] < past[:, None, None, None],
                                      caches[0].float() * caches[2].unsqueeze(-1), 0.0).to(dt))


@pytest.mark.parametrize("heads", [(4, 4), (32, 2)])
def test_captured_steps(heads):
    """Two graphs of a step, replayed in turn with other inputs and lengths, give what eager calls give:
    no workspace is shared, nothing of a capture's lengths is kept."""
    B, V, D, N, T = 2, 500, 64, 900, len(TREE)
    g = torch.Generator(device="cuda").manual_seed(5)
    toy, caches = _state(F16, B, V, *heads, D, N, g)
    k, v = (torch.randn(B, heads[1], N, D, generator=g, device="cuda").half() for _ in range(2))
    fpkern.cache_write_q8(k, v, *caches, torch.zeros(B, dtype=torch.int32, device="cuda"))
    parents = torch.tensor(TREE, dtype=torch.int32, device="cuda")
    ins = [dict(tokens=torch.zeros(B, T, dtype=torch.int32, device="cuda"), past=torch.zeros(B, dtype=torch.int32, device="cuda"),
                uniform=torch.zeros(B, T, device="cuda"), draft=torch.full((B, T, V), 1.0 / V, device="cuda")) for _ in range(2)]
    mine = [tuple(t.clone() for t in caches) for _ in range(2)]
    run = lambda i, c: step(toy, c, ins[i]["tokens"], parents, ins[i]["past"], ins[i]["uniform"], ins[i]["draft"])  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(2):
            run(i, mine[i])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(run(i, mine[i]))
    for n in range(3):
        for i in range(2):
            ins[i]["tokens"].copy_(torch.randint(0, V, (B, T), generator=g, device="cuda"))
            ins[i]["past"].copy_(torch.randint(0, N - T, (B,), generator=g, device="cuda"))
            ins[i]["uniform"].copy_(torch.rand(B, T, generator=g, device="cuda") * 0.1)
        plain = [tuple(t.clone() for t in c) for c in mine]
        for i in (0, 1):
            graphs[i].replay()
        for i in (1, 0):
            want = run(i, plain[i])
            for a, b in zip(outs[i] + mine[i], want + plain[i]):
                assert torch.equal(a, b)
    assert fpkern.poll_status() == 0


def test_calls_on_other_streams_and_threads():
    """Calls of two threads, each on its own stream, beside one another."""
    import threading

    g = torch.Generator(device="cuda").manual_seed(6)
    B, H, Hk, T, N, D = 2, 16, 2, 12, 3000, 128
    q = torch.randn(B, H, T, D, generator=g, device="cuda").half()
    k, v = (torch.randn(B, Hk, N, D, generator=g, device="cuda") for _ in range(2))
    (k8, ks), (v8, vs) = quantised(k), quantised(v)
    parents = (torch.arange(T, device="cuda") - 1).to(torch.int32)
    past = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([2900, 50], [1000, 2000])]
    call = lambda i: fpkern.tree_attention(q, k8, v8, 0.09, parents, past[i], k_scale=ks, v_scale=vs)  # noqa: E731
    want = [call(i) for i in range(2)]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                if not torch.equal(call(i), want[i]):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not bad


def test_prompt_in_pieces_over_an_8_bit_cache():
    """A prompt written and attended to piece by piece: the cache read back for score_attention."""
    g = torch.Generator(device="cuda").manual_seed(7)
    B, H, Hk, N, D = 1, 4, 2, 300, 64
    q, k, v = (torch.randn(B, h, N, D, generator=g, device="cuda").half() for h in (H, Hk, Hk))
    caches = _state(F16, B, 8, H, Hk, D, N, g)[1]
    outs = []
    for at in range(0, N, 100):
        part = lambda t: t[:, :, at:at + 100]  # noqa: E731
        past, lens = (torch.tensor([x], dtype=torch.int32, device="cuda") for x in (at, at + 100))
        fpkern.cache_write_q8(part(k), part(v), *caches, past)
        kk, vv = fpkern.cache_read_q8(*caches, dtype=F16, kv_lens=lens)
        outs.append(fpkern.score_attention(part(q), kk, vv, 0.125, causal=True, kv_lens=lens))
    (k8, ks), (v8, vs) = quantised(k), quantised(v)
    whole = fpkern.score_attention(q, (k8 * ks.unsqueeze(-1)).half(), (v8 * vs.unsqueeze(-1)).half(), 0.125, causal=True)
    torch.testing.assert_close(torch.cat(outs, 2), whole, rtol=4e-3, atol=4e-3)
