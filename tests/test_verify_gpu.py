"""Which drafted tokens stay, on the GPU, against the walk in fp64 on the host: the same nodes and the same tokens."""
import math

import pytest
import torch

from prometorch_b200.ops.verify import verify_drafts, verify_drafts_reference

pytestmark = pytest.mark.gpu
DEV = "cuda"


def peaked(g, B, T, V):
    """Four tokens of each row carry most of it."""
    x = torch.randn(B, T, V, generator=g) * 1.5
    if V > 8:
        x.scatter_add_(2, torch.randint(0, V, (B, T, 4), generator=g), (torch.tensor([1.5, 0.5, -0.5, -1.5]) + math.log(V)).expand(B, T, 4))
    return x


def drafts(g, logits, parents):
    """Tokens drawn from the target at the parent, one in four at random."""
    B, T, V = logits.shape
    at = logits.gather(1, parents.long().clamp_min(0)[..., None].expand(B, T, V))
    noise = -torch.log(-torch.log(torch.rand(B, T, V, generator=g).clamp(1e-7, 1 - 1e-7)))
    tok = (at + noise).argmax(-1)
    return torch.where(torch.rand(B, T, generator=g) < 0.25, torch.randint(0, V, (B, T), generator=g), tok).int()


def check(logits, tokens, u, temperature, **kw):
    on = lambda t: t.to(DEV) if t is not None else None  # noqa: E731
    got = verify_drafts(on(logits), on(tokens), on(u), on(temperature), **{k: on(t) for k, t in kw.items()})
    want = verify_drafts_reference(logits, tokens, u, temperature, **kw)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b), (a.cpu(), b)
    return want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,V", [(1, 1, 1), (3, 4, 7), (5, 64, 500), (9, 17, 4097), (4, 9, 32000), (2, 5, 151936), (1, 2, 230000)])
def test_trees(dtype, B, T, V):
    g = torch.Generator().manual_seed(V + T)
    logits = peaked(g, B, T, V).to(dtype)
    i = torch.arange(T).repeat(B, 1)
    parents = torch.where(i > 0, (i - torch.randint(1, 6, (B, T), generator=g)).clamp_min(0), -1).int()
    tokens, u = drafts(g, logits.float(), parents), torch.rand(B, T, generator=g)
    temperature = torch.tensor([(1.0, 0.0, 0.6, -1.0, 2.5)[b % 5] for b in range(B)])
    nodes = torch.randint(0, T + 1, (B,), generator=g).int()
    nodes[0] = T
    path, count, _ = check(logits, tokens, u, temperature, parents=parents, nodes=nodes)
    if B == 9:                                   # these drafts are accepted several deep
        assert int(count.max()) >= 3
    check(logits, tokens, u, temperature)


@pytest.mark.parametrize("B,T,V", [(3, 3, 11), (6, 6, 4096), (5, 8, 32000), (2, 4, 151936)])
def test_chains_with_probabilities(B, T, V):
    g = torch.Generator().manual_seed(V)
    logits = peaked(g, B, T, V)
    near = logits + 0.7 * torch.randn(B, T, V, generator=g)
    probs = torch.softmax(near, -1)
    parents = torch.arange(-1, T - 1).repeat(B, 1)
    tokens, u = drafts(g, near, parents), torch.rand(B, T, generator=g)
    temperature = torch.tensor([(1.0, 1.0, 0.7, 0.0)[b % 4] for b in range(B)])
    check(logits, tokens, u, temperature, draft_probs=probs)
    # rows further apart, and a draft that is the target itself: everything is accepted
    wide = torch.zeros(B, T, V + 5)
    wide[..., 2:2 + V] = logits
    on = lambda t: t.to(DEV)  # noqa: E731
    one = torch.ones(B)
    got = verify_drafts(on(wide)[..., 2:2 + V], on(tokens), on(u * 0.999), on(one), draft_probs=on(torch.softmax(logits.double(), -1).float()))
    assert got[1].tolist() == [T - 1] * B


def test_masked_logits_equal_siblings_and_strange_tokens():
    g = torch.Generator().manual_seed(4)
    B, T, V = 8, 6, 1000
    logits = peaked(g, B, T, V)
    logits[0] = -math.inf                        # nothing has a probability
    logits[1, :, 1:] = -math.inf                 # one token has it all
    logits[2, :, ::2] = math.nan
    logits[3, 0, 5] = logits[3, 0, 9] = math.inf
    logits[4] = 1.0                              # all equal
    parents = torch.tensor([[-1, 0, 0, 0, 1, 3]] * B, dtype=torch.int32)
    parents[7] = torch.tensor([-1, 0, 2, 5, -1, 1])          # a node that is its own parent, one behind its child, one without any
    tokens = drafts(g, logits.nan_to_num(0, 0, 0), parents)
    tokens[5, 1:4] = tokens[5, 1].clone()        # siblings with one token
    tokens[6, 1], tokens[6, 2] = -3, V
    for seed in range(6):
        h = torch.Generator().manual_seed(seed)
        u = torch.rand(B, T, generator=h) if seed else torch.zeros(B, T)
        for t in (1.0, 0.0, 0.3):
            check(logits, tokens, u, torch.full((B,), t), parents=parents)


def test_tokens_are_distributed_as_the_target():
    """20000 requests with the same logits: the first token that comes out, whether a draft or not, has the target's probabilities (within five standard deviations)."""
    V, B, rounds = 12, 5000, 4
    g = torch.Generator(device=DEV).manual_seed(1)
    row = torch.randn(V, generator=g, device=DEV) * 1.5
    p = torch.softmax(row.double(), 0)
    q = torch.softmax(row + torch.randn(V, generator=g, device=DEV), 0)
    one = torch.ones(B, device=DEV)
    for tree in (False, True):
        seen = torch.zeros(V, dtype=torch.float64, device=DEV)
        for _ in range(rounds):
            T = 4 if tree else 2
            logits = row.expand(B, T, V)
            u = torch.rand(B, T, generator=g, device=DEV)
            if tree:       # three siblings with tokens of their own, proposed outright
                tokens = torch.tensor([0, 3, 7, 1], dtype=torch.int32, device=DEV).repeat(B, 1)
                parents = torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device=DEV).repeat(B, 1)
                _, _, out = verify_drafts(logits, tokens, u, one, parents=parents)
            else:
                tokens = torch.multinomial(q, B * T, replacement=True, generator=g).view(B, T).int()
                _, _, out = verify_drafts(logits, tokens, u, one, draft_probs=q.expand(B, T, V).contiguous())
            seen += torch.bincount(out[:, 0].long(), minlength=V)
        n = B * rounds
        assert bool(((seen / n - p).abs() <= 5 * torch.sqrt(p * (1 - p) / n)).all()), (tree, seen / n, p)


def test_streams_graphs_and_repeats():
    g = torch.Generator().manual_seed(2)
    B, T, V = 4, 8, 5000
    logits = peaked(g, B, T, V).to(DEV)
    parents = torch.tensor([[-1, 0, 0, 1, 2, 3, 3, 5]] * B, dtype=torch.int32)
    args = [logits, drafts(g, logits.cpu(), parents).to(DEV), torch.rand(B, T, generator=g).to(DEV), torch.ones(B, device=DEV)]
    dev_parents = parents.to(DEV)
    call = lambda: verify_drafts(*args, parents=dev_parents)  # noqa: E731
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(call())
        graphs.append(gr)
    args[2].copy_(torch.rand(B, T, generator=g))
    for gr in graphs:
        gr.replay()
    want = call()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t", [math.inf, 3e38, 1e38, 2e30, 0.9e30, 1e4, 1e-3, 1.2e-38, math.nan])
def test_temperatures_of_any_size(dtype, t):
    """A row is as good as uniform, or as good as its arg-max; masked logits (-inf, the type's lowest value) and the end of the last chunk behind the vocabulary are what they are at any other."""
    g = torch.Generator().manual_seed(6)
    B, T, V = 6, 8, 9001
    logits = peaked(g, B, T, V)
    logits[1, :, ::3] = -math.inf
    logits[2, :, 5:] = -math.inf
    logits[3, :, 1::2] = torch.finfo(dtype).min
    logits[4, :, ::2] = 3e38
    logits[5, 0, 7] = math.inf
    parents = torch.tensor([[-1, 0, 0, 0, 1, 1, 2, 4]] * B, dtype=torch.int32)
    logits, tokens = logits.to(dtype), torch.randint(0, V, (B, T), generator=g).int()
    tokens[2] %= 5
    tokens[:, 1] = logits[:, 0].float().argmax(-1).int()
    for seed in range(3):
        u = torch.rand(B, T, generator=torch.Generator().manual_seed(seed))
        u[:, 1:] *= (1.0, 1.0, 1e-4)[seed]                # small numbers accept tokens of a uniform row
        check(logits, tokens, u, torch.full((B,), t), parents=parents)
        check(logits, tokens, u, torch.full((B,), t))


@pytest.mark.parametrize("B,T", [(1024, 64), (65535, 1), (8192, 8)])
def test_as_many_nodes_as_the_attention_takes(B, T):
    g = torch.Generator().manual_seed(T)
    V = 5
    logits = torch.randn(B, T, V, generator=g)
    parents = (torch.arange(T).repeat(B, 1) - torch.randint(1, 4, (B, T), generator=g)).clamp_min(-1).int()
    tokens, u = torch.randint(0, V, (B, T), generator=g).int(), torch.rand(B, T, generator=g)
    args = [t.to(DEV) for t in (logits, tokens, u, torch.ones(B))]
    got = verify_drafts(*args, parents=parents.to(DEV))
    assert int(got[1].min()) >= 0 and bool((got[2] < V).all())
    some = torch.cat([torch.arange(40), torch.arange(B - 200, B)])
    want = verify_drafts_reference(logits[some], tokens[some], u[some], torch.ones(240), parents=parents[some])
    for a, b in zip(got, want):
        assert torch.equal(a.cpu()[some], b)
    with pytest.raises(RuntimeError, match="in all"):
        verify_drafts(torch.zeros(B + 1, T, V, device=DEV), torch.zeros(B + 1, T, dtype=torch.int32, device=DEV), torch.zeros(B + 1, T, device=DEV), torch.zeros(B + 1, device=DEV))
