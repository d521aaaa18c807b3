"""GPU: the verification of drafted tokens against its definition, whole numbers equal."""

import pytest
import torch

from fusionpass_b200 import fpkern
from tests._draft_ref import verify_reference

pytestmark = pytest.mark.gpu


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _inputs(B, T, V, g, noise=0.7):
    logits = 2.0 * torch.randn(B, T, V, generator=g, device="cuda")
    target = torch.softmax(logits, -1)
    draft = torch.softmax(logits + noise * torch.randn(B, T, V, generator=g, device="cuda"), -1)
    i = torch.arange(T, device="cuda")
    parents = (torch.rand(B, T, generator=g, device="cuda") * i * 0.7).long()
    parents[:, 0] = -1
    drawn = torch.multinomial(draft.reshape(B * T, V), T, replacement=True, generator=g).reshape(B, T, T)
    tokens = drawn.gather(1, parents.clamp(min=0)[..., None].expand(B, T, T)).gather(2, i.expand(B, T)[..., None])[..., 0]
    uniform = torch.rand(B, T, generator=g, device="cuda")
    return tokens.to(torch.int32), parents.to(torch.int32), target, draft, uniform


def check(tokens, parents, target, draft, uniform, lens=None):
    B, T = tokens.shape
    full = parents if parents.dim() == 2 else parents.expand(B, T)
    want = verify_reference(tokens, full, target, draft, uniform, lens if lens is not None else [T] * B)
    got = fpkern.verify_draft(tokens, parents, target, draft, uniform, tree_lens=lens)
    for a, b in zip(got, want):
        assert a.dtype == torch.int32 and torch.equal(a.cpu(), b), (a, b)
    return got


# V around a stretch of 32, 512 (a CTA's warps), 4096 (one CTA), and several CTAs
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 1, 7), (3, 5, 31), (2, 9, 33), (40, 6, 511), (5, 40, 513), (3, 12, 4096),
                                   (4, 8, 4097), (2, 20, 20000), (6, 33, 50001), (1, 8, 32000), (2, 70, 9001),
                                   (200, 4, 5000), (3, 256, 300)])
@pytest.mark.parametrize("with_draft", [True, False])
def test_against_definition(with_draft, shape):
    B, T, V = shape
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    tokens, parents, target, draft, uniform = _inputs(B, T, V, g)
    lens = torch.randint(0, T + 2, (B,), generator=g, device="cuda").to(torch.int32)
    draft = draft if with_draft else None
    path, counts, nxt = check(tokens, parents, target, draft, uniform)
    assert (counts >= 1).all() and (nxt >= 0).all() and (nxt < V).all()
    check(tokens, parents, target, draft, uniform, lens)
    check(tokens, parents[0].contiguous(), target, draft, uniform, lens)


def test_many_failures_at_one_node():
    """A star of drafts that fail one after another, tokens twice among them; then the last stands."""
    B, T, V = 8, 200, 3000
    g = torch.Generator(device="cuda").manual_seed(2)
    tokens, _, target, draft, uniform = _inputs(B, T, V, g, noise=3.0)
    parents = torch.where(torch.arange(T, device="cuda") > 0, 0, -1).to(torch.int32)
    tokens[:, 50:100] = tokens[:, 1:51]
    uniform[:, 1:] = 0.999
    for d in (draft, None):
        check(tokens, parents, target, d, uniform)
    uniform[:, 150] = 0.0
    for d in (draft, None):
        path, counts, _ = check(tokens, parents, target, d, uniform)


def test_certain_cases():
    """Draft and target alike: all of a chain stands.  Nothing in common: the first fails, and the next
    token is the target's.  Numbers at the ends of [0, 1)."""
    B, T, V = 4, 6, 1000
    chain = (torch.arange(T, device="cuda") - 1).to(torch.int32)
    g = torch.Generator(device="cuda").manual_seed(3)
    tokens, _, target, _, uniform = _inputs(B, T, V, g)
    at = torch.multinomial(target.reshape(B * T, V), 1, generator=g).reshape(B, T)
    tokens[:, 1:] = at[:, :-1]
    path, counts, nxt = check(tokens, chain, target, target, uniform)
    assert counts.eq(T).all() and torch.equal(path, torch.arange(T, device="cuda").int().expand(B, T))
    p, q = target.clone(), target.clone()
    p[..., ::2], q[..., 1::2] = 0.0, 0.0
    p, q = p / p.sum(-1, keepdim=True), q / q.sum(-1, keepdim=True)
    tokens[:, 1:] = tokens[:, 1:] // 2 * 2
    path, counts, nxt = check(tokens, chain, p, q, uniform)
    assert counts.eq(1).all() and (nxt % 2 == 1).all()
    for u in (0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, float("nan")):
        full = torch.full((B, T), u, device="cuda")
        for d in (target, q, None):
            check(tokens, chain, target, d, full)


def test_borders():
    """Probabilities of whole powers of two: running sums are exact, numbers fall on borders."""
    V = 1024
    target = torch.full((64, 1, V), 1.0 / V, device="cuda")
    u = (torch.arange(64, device="cuda") / 64.0)[:, None]
    _, _, nxt = check(torch.zeros(64, 1, dtype=torch.int32, device="cuda"), i32(-1), target, None, u)
    assert torch.equal(nxt.cpu(), (torch.arange(64) * 16).int())


def test_probabilities_that_are_not_ordinary():
    g = torch.Generator(device="cuda").manual_seed(4)
    for V in (40, 6000):
        tokens, parents, target, draft, uniform = _inputs(9, 8, V, g)
        target[0] = 0.0
        target[1] = float("nan")
        target[2, :, 3] = float("inf")
        target[3] = -1.0
        target[4, :, ::2] = float("nan")
        target[5, 0] = 0.0
        target[5, 0, V - 1] = 1e-42
        draft[6] = 0.0
        draft[7] = float("nan")
        tokens[8, ::2] = V
        tokens[8, 1] = -1
        for d in (draft, None):
            path, counts, nxt = check(tokens, parents, target, d, uniform)
            assert nxt[:4].tolist() == [-1, -1, -1, -1] or d is not None


def test_parents_that_are_no_earlier_node():
    g = torch.Generator(device="cuda").manual_seed(5)
    tokens, parents, target, draft, uniform = _inputs(6, 10, 300, g)
    parents[:, 3], parents[:, 4], parents[:, 5] = 3, 9, -7
    parents[0] = 0
    parents[1] = 2147483647
    check(tokens, parents, target, draft, uniform)


def test_strides():
    """Rows of a padded vocabulary, nodes' rows of another order, one number table for all."""
    B, T, V = 3, 5, 1001
    g = torch.Generator(device="cuda").manual_seed(6)
    tokens, parents, target, draft, uniform = _inputs(B, T, V, g)
    want = check(tokens, parents, target, draft, uniform)
    wide = torch.full((T, B, V + 23), float("nan"), device="cuda")
    wide[..., 23:] = target.transpose(0, 1)
    rest = draft.transpose(1, 2).contiguous().transpose(1, 2)
    got = fpkern.verify_draft(tokens.t().contiguous().t(), parents, wide[..., 23:].transpose(0, 1), rest, uniform)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_a_vocabulary_of_the_largest_size():
    g = torch.Generator(device="cuda").manual_seed(7)
    V = 1 << 22
    tokens, parents, target, draft, uniform = _inputs(1, 3, V, g)
    check(tokens, parents, target, draft, uniform)
    check(tokens, parents, target, None, uniform)


def test_rows_beyond_32_bits():
    """The last row starts behind 2^31 elements."""
    T, V = 17, 1 << 17
    B = (1 << 31) // (T * V) + 1
    target = torch.zeros(B, T, V, device="cuda")
    target[B - 1, T - 1, 77] = 1.0
    target[B - 1, 0, 5] = 1.0
    tokens = torch.zeros(B, T, dtype=torch.int32, device="cuda")
    tokens[B - 1, T - 1] = 5
    parents = torch.where(torch.arange(T, device="cuda") == T - 1, 0, -1).to(torch.int32)
    path, counts, nxt = fpkern.verify_draft(tokens, parents, target, None, torch.full((B, T), 0.5, device="cuda"))
    assert path[B - 1, :3].tolist() == [0, T - 1, -1] and counts[B - 1] == 2 and nxt[B - 1] == 77 and nxt[0] == -1


@pytest.mark.parametrize("with_draft", [True, False])
def test_the_first_token_is_distributed_as_the_target(with_draft):
    """One draft and all of a grid of numbers: a token's share is its probability, up to the grid (a border
    of each of the two numbers: 2 cells a row or column of 128)."""
    V, n = 6, 128
    g = torch.Generator(device="cuda").manual_seed(8)
    p, q = (torch.softmax(torch.randn(V, generator=g, device="cuda"), 0) for _ in range(2))
    grid = (torch.arange(n, device="cuda") + 0.5) / n
    u = torch.cartesian_prod(grid, grid)
    B = u.shape[0]
    share = torch.zeros(V, dtype=torch.float64, device="cuda")
    for x in range(V):
        tokens = torch.tensor([[0, x]], dtype=torch.int32, device="cuda").expand(B, 2)
        rows = lambda t: t.expand(B, 2, V)  # noqa: E731
        path, counts, nxt = fpkern.verify_draft(tokens, i32(-1, 0), rows(p), rows(q) if with_draft else None, u)
        first = torch.where(counts == 2, x, nxt).long()
        weight = q[x].double() if with_draft else 1.0 / V
        share += weight * torch.bincount(first, minlength=V) / B
    assert (share - p.double()).abs().max() <= 4.0 / n


def test_empty_and_refused_calls():
    g = torch.Generator(device="cuda").manual_seed(9)
    tokens, parents, target, draft, uniform = _inputs(2, 4, 50, g)
    f = fpkern.verify_draft
    path, counts, nxt = f(tokens[:0], parents[:0], target[:0], draft[:0], uniform[:0])
    assert path.shape == (0, 4) and counts.shape == nxt.shape == (0,)
    bad = [
        lambda: f(tokens.long(), parents, target, draft, uniform),
        lambda: f(tokens[0], parents, target, draft, uniform),
        lambda: f(tokens, parents.long(), target, draft, uniform),
        lambda: f(tokens, parents[:, :3], target, draft, uniform),
        lambda: f(tokens, parents, target.half(), draft, uniform),
        lambda: f(tokens, parents, target[:, :3], draft, uniform),
        lambda: f(tokens, parents, target[..., :0], None, uniform),
        lambda: f(tokens, parents, target, draft[..., :49], uniform),
        lambda: f(tokens, parents, target, draft.double(), uniform),
        lambda: f(tokens, parents, target, draft, uniform.double()),
        lambda: f(tokens, parents, target, draft, uniform[:1]),
        lambda: f(tokens, parents, target, draft, uniform, tree_lens=i32(1)),
        lambda: f(tokens[:, :0], parents[:, :0], target[:, :0], None, uniform[:, :0]),
        lambda: f(tokens.repeat(1, 65), parents.repeat(1, 65), target.repeat(1, 65, 1), None, uniform.repeat(1, 65)),
        lambda: f(tokens, parents, target.clone().requires_grad_(), draft, uniform),
        lambda: f(tokens, parents, torch.zeros(1, 1, 1, device="cuda").expand(2, 4, (1 << 22) + 1), None, uniform),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(RuntimeError):
        f(tokens, parents, target.cpu(), draft, uniform)
