"""Which drafted tokens stay: the walk on the host against hand-made cases and frequencies, and what is refused."""
import math

import pytest
import torch

from prometorch_b200.ops.verify import verify_drafts

BASE = 1 << 20


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def from_probs(*rows):
    return torch.log(torch.tensor(rows))[None]


def test_a_tree_by_hand():
    logits = from_probs([0.5, 0.3, 0.2], [0.1, 0.1, 0.8], [1 / 3, 1 / 3, 1 / 3], [0.0, 1.0, 0.0])
    tokens, parents = i32(9, 0, 1, 2)[None], i32(-1, 0, 0, 1)[None]
    one = torch.ones(1)
    # child 1 (p 0.5) accepted, its child 3 (p 0.8) accepted, the last token is certain
    path, count, out = verify_drafts(logits, tokens, torch.tensor([[0.3, 0.49, 0.9, 0.79]]), one, parents=parents)
    assert path.tolist() == [[0, 1, 3, -1]] and count.tolist() == [2] and out.tolist() == [[0, 2, 1, -1]]
    # child 1 rejected; child 2 has 0.3 of the 0.5 that are left
    path, count, out = verify_drafts(logits, tokens, torch.tensor([[0.5, 0.51, 0.59, 0.0]]), one, parents=parents)
    assert path.tolist() == [[0, 2, -1, -1]] and out.tolist() == [[1, 1, -1, -1]]
    # both rejected: only token 2 is left
    path, count, out = verify_drafts(logits, tokens, torch.tensor([[0.0, 0.51, 0.61, 0.0]]), one, parents=parents)
    assert path.tolist() == [[0, -1, -1, -1]] and count.tolist() == [0] and out.tolist() == [[2, -1, -1, -1]]
    # greedy: the arg-max of each row
    path, count, out = verify_drafts(logits, tokens, torch.zeros(1, 4), torch.zeros(1), parents=parents)
    assert path.tolist() == [[0, 1, 3, -1]] and out.tolist() == [[0, 2, 1, -1]]


def test_a_chain_with_probabilities_by_hand():
    logits, q = from_probs([0.5, 0.3, 0.2], [0.2, 0.2, 0.6]), torch.tensor([[[0.2, 0.7, 0.1], [1 / 3, 1 / 3, 1 / 3]]])
    one, tokens = torch.ones(1), i32(0, 1)[None]
    # token 1: p 0.3, q 0.7
    assert verify_drafts(logits, tokens, torch.tensor([[0.3, 0.42]]), one, draft_probs=q)[2].tolist() == [[1, 1]]
    # rejected: max(p - q, 0) is 0.3 and 0.1 for tokens 0 and 2
    assert verify_drafts(logits, tokens, torch.tensor([[0.74, 0.43]]), one, draft_probs=q)[2].tolist() == [[0, -1]]
    assert verify_drafts(logits, tokens, torch.tensor([[0.76, 0.43]]), one, draft_probs=q)[2].tolist() == [[2, -1]]


def test_nothing_to_draw_from_and_no_nodes():
    logits = torch.full((2, 2, 4), -math.inf)
    path, count, out = verify_drafts(logits, i32(0, 0, 0, 0).view(2, 2), torch.rand(2, 2), torch.ones(2), nodes=i32(2, 0))
    assert out.tolist() == [[0, -1], [-1, -1]] and count.tolist() == [0, -1] and path.tolist() == [[0, -1], [-1, -1]]


@pytest.mark.parametrize("tree", [False, True])
def test_the_target_s_distribution_comes_out(tree):
    """Within five standard deviations of 4000 draws."""
    V, B = 5, 4000
    g = torch.Generator().manual_seed(0)
    row = torch.randn(V, generator=g)
    p, q = torch.softmax(row.double(), 0), torch.softmax(torch.randn(V, generator=g), 0)
    T = 3 if tree else 2
    logits, u, one = row.expand(B, T, V), torch.rand(B, T, generator=g), torch.ones(B)
    if tree:
        out = verify_drafts(logits, i32(0, 3, 1).repeat(B, 1), u, one, parents=i32(-1, 0, 0).repeat(B, 1))[2]
    else:
        out = verify_drafts(logits, torch.multinomial(q, B * T, replacement=True, generator=g).view(B, T).int(), u, one, draft_probs=q.expand(B, T, V))[2]
    seen = torch.bincount(out[:, 0].long(), minlength=V) / B
    assert bool(((seen - p).abs() <= 5 * torch.sqrt(p * (1 - p) / B)).all())


def test_refusals():
    ok = dict(logits=torch.randn(2, 3, 7), tokens=torch.zeros(2, 3, dtype=torch.int32), u=torch.rand(2, 3), temperature=torch.ones(2))
    verify_drafts(**ok)
    for bad in (dict(logits=torch.randn(2, 3, 7).double()), dict(logits=torch.randn(6, 7)), dict(logits=torch.randn(2, 65, 7)), dict(tokens=torch.zeros(2, 3, dtype=torch.long)),
                dict(u=torch.rand(2, 2)), dict(temperature=torch.ones(2).double()), dict(parents=torch.zeros(2, 2, dtype=torch.int32)), dict(nodes=torch.zeros(3, dtype=torch.int32)),
                dict(draft_probs=torch.rand(2, 3, 8)), dict(draft_probs=torch.rand(2, 3, 7), parents=torch.zeros(2, 3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            verify_drafts(**{**ok, **bad})


def test_native_entry_refuses():
    from prometorch_b200 import _native as N
    L = N.lib()

    def call(B=2, T=3, V=100, probs=None, parents=None, work=BASE):
        rc = L.ptb_verify_drafts(BASE, 0, 300, 100, probs, 300, 100, BASE, parents, None, BASE, BASE, work, BASE, BASE, BASE, B, T, V, None)
        return rc == -1 and L.ptb_last_error().decode() or ""
    assert "nodes" in call(T=65) and "nodes" in call(T=0) and "tokens" in call(V=1 << 20) and "in all" in call(B=20000, T=8)
    assert "chains" in call(probs=BASE, parents=BASE) and "aligned" in call(work=BASE + 8)


def test_an_infinite_temperature():
    """Every token that has a probability has the same; of infinite logits only they have one."""
    V, inf = 6, math.inf
    logits = torch.tensor([[0.0, -inf, 3.0, 1.0, -inf, -2.0], [inf, 1.0, -inf, inf, 0.0, 0.0]])[:, None]
    for u, want in ((0.0, [0, 0]), (0.26, [2, 0]), (0.51, [3, 3]), (0.99, [5, 3])):
        out = verify_drafts(logits, torch.zeros(2, 1, dtype=torch.int32), torch.full((2, 1), u), torch.full((2,), inf))[2]
        assert out.flatten().tolist() == want
