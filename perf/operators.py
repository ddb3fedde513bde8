"""What speculative decoding over a paged cache does between two passes of a model, timed by itself: the cache entries of drafted tokens written (as they
are or quantised), attention of a tree of drafted tokens over the cache, the decision which of them stay, and the entries of those moved into place.

Four kinds of case, named by ``op``:

* ``write``: the packed projection of ``n`` tokens of ``batch`` sequences; q and k are rotated, k and v go to their slots of 64-token pages, in bf16 or
  in e4m3 with a power-of-two exponent for each token and head;
* ``attend``: ``nodes`` drafted tokens of each of ``batch`` requests over up to ``longest`` cached ones (half as many at least) and their ancestors among the drafted
  ones; one node is the plain decode step;
* ``verify``: the target's logits at every drafted token, the draft's probabilities for a chain (or a tree of tokens without any), uniform numbers;
* ``keep``: the accepted path of every request, its entries moved to the front of the drafted ones in every layer's pages.

Heads, head sizes and vocabularies are those of the benchmarks (``bench.py``, ``benchmarks/``).  Inputs are random; what is cached has unit variance with
a few larger channels, as keys do."""
import math

import torch

own = False
PAGE = 64
E4M3, LARGEST = torch.float8_e4m3fn, 448.0
LLAMA_1B, LLAMA_7B, QWEN_4B = (32, 4, 64), (32, 32, 128), (32, 8, 128)          # heads, kv heads, head size
VOCABS = (32000, 151936)


def _write(name, n, batch, heads, kind, want_k):
    return dict(name=name, op="write", n=n, batch=batch, heads=heads[0], kv_heads=heads[1], head_dim=heads[2], kind=kind, want_k=want_k)


def _attend(name, batch, nodes, longest, heads, kind, tree):
    return dict(name=name, op="attend", batch=batch, nodes=nodes, longest=longest, heads=heads[0], kv_heads=heads[1], head_dim=heads[2], kind=kind, tree=tree)


def _verify(name, batch, nodes, vocab, dtype, drafted):
    return dict(name=name, op="verify", batch=batch, nodes=nodes, vocab=vocab, dtype=dtype, drafted=drafted)


def _keep(name, layers, batch, nodes, heads, kind):
    return dict(name=name, op="keep", layers=layers, batch=batch, nodes=nodes, kv_heads=heads[1], head_dim=heads[2], kind=kind)


def listed():
    return [
        # one request and its eight drafted tokens, a quantised cache: a launch
        _write("write-8-e4m3", 8, 1, QWEN_4B, "e4m3", False),
        # a batch of trees of no round size into a plain cache, positions apart from slots
        _write("write-416-bf16", 416, 32, LLAMA_1B, "bf16", False),
        # the prompts of a batch, as many tokens as the engine lets share a pass, quantised on their way into the cache
        _write("write-16384-e4m3", 16384, 8, LLAMA_7B, "e4m3", True),
        # one user, a chain of four drafted tokens behind a short conversation
        _attend("attend-chain-5", 1, 5, 540, QWEN_4B, "bf16", False),
        # the plain decode step of a batch over a quantised cache
        _attend("attend-decode-32", 32, 1, 2040, LLAMA_1B, "e4m3", False),
        # a batch of trees over a quantised cache
        _attend("attend-tree-16", 16, 16, 4100, QWEN_4B, "e4m3", True),
        # wide trees over a plain cache: products count
        _attend("attend-tree-64", 8, 64, 8191, LLAMA_1B, "bf16", True),
        # a chain behind one very long document
        _attend("attend-long-8", 1, 8, 131071, QWEN_4B, "e4m3", False),
        # a batch of chains with a draft model's probabilities
        _verify("verify-chain-5", 8, 5, 32000, "fp32", True),
        # a batch of trees over a large vocabulary
        _verify("verify-tree-16", 32, 16, 151936, "fp32", False),
        # one user's accepted tokens in every layer of a 4B-class model, quantised
        _keep("keep-1", 36, 1, 8, QWEN_4B, "e4m3"),
        # those of a batch of trees
        _keep("keep-32", 32, 32, 16, QWEN_4B, "bf16"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "attend", "attend", "verify", "keep"])
    kind = rng.choice(["bf16", "e4m3"])
    if op == "write":
        kv = rng.choice([2, 4, 8, 32])
        group = 1 if kv == 32 else rng.choice([1, 2, 4, 8])
        n = _spread(rng, 1, 16384)
        c = _write("", n, rng.randint(1, min(n, 32)), (kv * group, kv, rng.choice([64, 128])), kind, rng.random() < 0.5)
    elif op == "attend":
        kv, nodes, size = rng.choice([2, 4, 8]), _spread(rng, 1, 64), rng.choice([64, 128])
        group = rng.choice([1, 2, 4, 8])
        batch, longest = _spread(rng, 1, 64), _spread(rng, 1, 131071)
        while batch * longest * kv * size * (1 + (kind == "bf16")) > 131071 * 8 * 128 or batch * longest * kv * group * nodes * size > 8 * 8191 * 32 * 64 * 64:
            batch, longest = max(1, batch // 2), max(1, longest * 2 // 3)
        c = _attend("", batch, nodes, longest, (kv * group, kv, size), kind, rng.random() < 0.5)
    elif op == "verify":
        batch, nodes, vocab = _spread(rng, 1, 64), _spread(rng, 1, 32), _spread(rng, 500, 151936)
        while batch * nodes * vocab > 32 * 16 * 151936:
            batch = max(1, batch // 2)
        c = _verify("", batch, nodes, vocab, rng.choice(["fp32", "bf16"]), rng.random() < 0.5)
    else:
        c = _keep("", rng.randint(1, 36), _spread(rng, 1, 32), _spread(rng, 1, 32), (0, rng.choice([2, 4, 8]), rng.choice([64, 128])), kind)
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------------------- inputs
def _quantise(x):
    """Values that e4m3 holds and the biased exponents: x = value * 2^(exponent - 127), one exponent for the last dimension."""
    m, k = torch.frexp(x.abs().amax(-1, keepdim=True))
    e = torch.where(m <= 0.875, k - 9, k - 8)                                       # the least with max |x| <= 448 * 2^e
    e = torch.where(m > 0, e, -64).clamp(-64, 64)
    return torch.ldexp(x, -e).clamp(-LARGEST, LARGEST).to(E4M3), (e + 127).to(torch.uint8).squeeze(-1)


def _stored(x, kind):
    """``x`` as a pool of that kind holds it: (values, exponents or None)."""
    return _quantise(x.float()) if kind == "e4m3" else (x.bfloat16(), None)


def _pools(g, n, kv, size, kind):
    """Keys and values of ``n`` pages: [k, k exponents, v, v exponents]."""
    def one(loud):
        parts = []
        for i in range(0, n, 4096):                                                 # 4096 pages at a time: the fp32 draw of a long cache is large
            x = torch.randn(min(4096, n - i), kv, PAGE, size, device="cuda", generator=g, dtype=torch.bfloat16)
            x[..., :loud] *= 4
            parts.append(_stored(x, kind))
        return [torch.cat(p) if p[0] is not None else None for p in zip(*parts)]
    return [*one(size // 32), *one(0)]


def _table(g, most):
    """Pages for up to ``most`` tokens each, in no order: (table [batch, most pages], pages in the pool)."""
    need = [max(1, -(-x // PAGE)) for x in most]
    order = torch.randperm(sum(need) + 1, generator=g)
    table, at = torch.zeros(len(most), max(need) + 1, dtype=torch.int32), 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    return table.cuda(), sum(need) + 1


def _parents(g, batch, nodes, tree):
    """Node i's parent, a node before it; -1 for the first, which is the latest token itself."""
    if not tree:
        return torch.arange(-1, nodes - 1, dtype=torch.int32).repeat(batch, 1)
    i = torch.arange(nodes).repeat(batch, 1)
    back = torch.randint(1, 7, (batch, nodes), generator=g)
    return torch.where(i > 0, (i - back).clamp_min(0), -1).int()


def _sees(parents):
    """[batch, node, node]: whether a node is the other or has it among its ancestors."""
    batch, nodes = parents.shape
    up = torch.zeros(batch, nodes, nodes, dtype=torch.float64, device=parents.device)
    up.scatter_(2, parents.long().clamp_min(0)[..., None], (parents >= 0).double()[..., None])
    return torch.linalg.matrix_power(up + torch.eye(nodes, dtype=torch.float64, device=parents.device), max(1, nodes)) > 0


def _bits(sees):
    return (sees.long() << torch.arange(sees.shape[-1], device=sees.device)).sum(-1)


def _counts(g, batch, nodes):
    """Nodes of every request: half of the tree at least, the first one's whole."""
    n = torch.randint((nodes + 1) // 2, nodes + 1, (batch,), generator=g)
    n[0] = nodes
    return n.int()


def prepare(case, seed):
    g, host = torch.Generator(device="cuda").manual_seed(seed), torch.Generator().manual_seed(seed)
    s = dict(case)
    if case["op"] == "write":
        n, batch, H, Hk, D = case["n"], case["batch"], case["heads"], case["kv_heads"], case["head_dim"]
        each = [n // batch + (b < n % batch) for b in range(batch)]
        starts = torch.randint(0, 500, (batch,), generator=host).tolist() if not case["want_k"] else [0] * batch
        pos, slot, req = [], [], []
        for b, k in enumerate(each):
            i = torch.arange(k)
            slot.append(starts[b] + i)
            pos.append(starts[b] + (i if case["want_k"] else (i + 1) // 2))         # a prompt, or drafted tokens two to a depth
            req.append(torch.full((k,), b))
        s["table"], pages = _table(host, [k if case["want_k"] else 500 + k for k in each])
        s["pos"], s["slot"], s["req"] = (torch.cat(t).int().cuda() for t in (pos, slot, req))
        s["k"], s["ke"], s["v"], s["ve"] = _pools(g, pages, Hk, D, case["kind"])
        s["qkv"] = torch.randn(n, (H + 2 * Hk) * D, device="cuda", generator=g).bfloat16()
        freq = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
        a = torch.arange(int(s["pos"].max()) + 1, dtype=torch.float64, device="cuda")[:, None] * freq
        s["cos"], s["sin"] = a.cos().float(), a.sin().float()
    elif case["op"] == "attend":
        B, T, H, Hk, D = case["batch"], case["nodes"], case["heads"], case["kv_heads"], case["head_dim"]
        lens = torch.randint((case["longest"] + 1) // 2, case["longest"] + 1, (B,), generator=host)
        lens[0] = case["longest"]
        s["count"], s["lens"] = _counts(host, B, T).cuda(), lens.int().cuda()
        s["table"], pages = _table(host, [case["longest"] + T] * B)
        s["k"], s["ke"], s["v"], s["ve"] = _pools(g, pages, Hk, D, case["kind"])
        s["mask"] = _bits(_sees(_parents(host, B, T, case["tree"]).cuda()))
        s["q"] = torch.randn(B, T, H * D, device="cuda", generator=g).bfloat16()
    elif case["op"] == "verify":
        B, T, V = case["batch"], case["nodes"], case["vocab"]
        logits = torch.randn(B, T, V, device="cuda", generator=g) * 1.5
        # four tokens of every distribution carry two thirds of it
        ids, more = torch.randint(0, V, (B, T, 4), device="cuda", generator=g), torch.tensor([1.5, 0.5, -0.5, -1.5], device="cuda") + math.log(V)
        logits.scatter_add_(2, ids, more.expand(B, T, 4))
        parents = _parents(host, B, T, not case["drafted"]).cuda()
        near = (logits + 0.7 * torch.randn(logits.shape, device="cuda", generator=g)) if case["drafted"] else logits
        noise = -torch.log(-torch.log(torch.rand(logits.shape, device="cuda", generator=g).clamp(1e-7, 1 - 1e-7)))
        at = parents.long().clamp_min(0)
        # drawn from the draft's distribution at the parent (or the target's), siblings each with noise of their own
        wanted = near.gather(1, at[..., None].expand(B, T, V))
        s["tokens"] = (wanted + noise).argmax(-1).int()
        s["probs"] = torch.softmax(near, -1) if case["drafted"] else None
        s["logits"] = logits.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
        s["parents"] = None if case["drafted"] else parents
        s["count"] = _counts(host, B, T).cuda()
        s["u"] = torch.rand(B, T, device="cuda", generator=g)
        s["temperature"] = torch.tensor([(1.0, 0.7, 0.0, 1.3)[b % 4] for b in range(B)], device="cuda")
    else:
        L, B, T, Hk, D = case["layers"], case["batch"], case["nodes"], case["kv_heads"], case["head_dim"]
        lens = torch.randint(1, 2000, (B,), generator=host)
        s["lens"] = lens.int().cuda()
        s["table"], pages = _table(host, [PAGE - 1 + T] * B)                           # the pages behind the whole ones
        wide = torch.zeros(B, 2000 // PAGE + 1 + s["table"].shape[1], dtype=torch.int32, device="cuda")
        cols = (s["lens"].long() // PAGE)[:, None] + torch.arange(s["table"].shape[1], device="cuda")
        s["table"] = wide.scatter_(1, cols, s["table"])
        # one tensor for all layers' keys and one for their values, of which the layers' pools are views
        stacks = [_pools(g, pages, Hk, D, case["kind"]) for _ in range(L)]
        s["k"], s["ke"], s["v"], s["ve"] = (torch.stack(t) if t[0] is not None else None for t in zip(*stacks))
        kept = torch.rand(B, T, generator=host) < 0.6
        kept[:, 0] = True
        order = torch.argsort((~kept).int(), dim=1, stable=True)
        n = kept.sum(1)
        s["path"] = torch.where(torch.arange(T) < n[:, None], order, -1).int().cuda()
        s["count"] = (n - 1).int().cuda()
        s["layers"] = list(zip(*(t.unbind(0) if t is not None else [None] * L for t in (s["k"], s["v"], s["ke"], s["ve"]))))
    return s


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(s):
    if s["op"] == "write":
        return _own_write(s) if own else _plain_write(s)
    if s["op"] == "attend":
        return _own_attend(s) if own else _plain_attend(s)
    if s["op"] == "verify":
        return _own_verify(s) if own else _plain_verify(s)
    return _own_keep(s) if own else _plain_keep(s)


def _own_write(s):
    from prometorch_b200.ops.paged_tree import paged_write
    q, k = paged_write(s["qkv"], s["heads"], s["kv_heads"], s["head_dim"], s["pos"], s["req"], s["table"], s["cos"], s["sin"], s["k"], s["v"], slot=s["slot"],
                       k_exp=s["ke"], v_exp=s["ve"], want_k=s["want_k"])
    return {"q": q, "k": k, "pages": [s["k"], s["v"], s["ke"], s["ve"]]}


def _plain_write(s):
    H, Hk, D = s["heads"], s["kv_heads"], s["head_dim"]
    x = s["qkv"].view(-1, H + 2 * Hk, D).float()
    c, sn = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]
    a, b = x[:, :H + Hk, :D // 2], x[:, :H + Hk, D // 2:]
    turned = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    slot = s["slot"].long()
    page, at = s["table"][s["req"].long(), slot // PAGE].long(), slot % PAGE
    ks, ke = _stored(turned[:, H:], s["kind"])
    vs, ve = _stored(x[:, H + Hk:], s["kind"])
    raw = (lambda t: t.view(torch.uint8)) if s["kind"] == "e4m3" else (lambda t: t)
    raw(s["k"])[page, :, at], raw(s["v"])[page, :, at] = raw(ks), raw(vs)
    if s["kind"] == "e4m3":
        s["ke"][page, :, at], s["ve"][page, :, at] = ke, ve
    return {"q": turned[:, :H].reshape(-1, H * D).bfloat16(), "k": turned[:, H:].bfloat16() if s["want_k"] else None, "pages": [s["k"], s["v"], s["ke"], s["ve"]]}


def _own_attend(s):
    from prometorch_b200.ops.paged_tree import paged_attention_tree
    return paged_attention_tree(s["q"], s["heads"], s["kv_heads"], s["head_dim"], s["lens"], s["table"], s["k"], s["v"], mask=s["mask"], nodes=s["count"],
                                k_exp=s["ke"], v_exp=s["ve"])


def _cached(pool, exps, table):
    """Keys or values of every request, [batch, kv heads, tokens, size] in fp32."""
    x = pool.view(torch.uint8)[table].view(E4M3).float() if exps is not None else pool[table].float()
    x = torch.ldexp(x, exps[table].int()[..., None] - 127) if exps is not None else x
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attend(s):
    B, T, H, Hk, D = s["batch"], s["nodes"], s["heads"], s["kv_heads"], s["head_dim"]
    table = s["table"][:, :-(-(s["longest"] + T) // PAGE)].long()
    k, v = _cached(s["k"], s["ke"], table), _cached(s["v"], s["ve"], table)
    at = torch.arange(k.shape[2], device="cuda") - s["lens"][:, None]                # a key's place among the nodes, negative for the cached ones
    bit = (s["mask"][:, :, None] >> at.clamp(0, 63)[:, None]) & 1
    sees = (at < 0)[:, None] | ((at < s["count"][:, None])[:, None] & (bit == 1))
    sees = sees & (torch.arange(T, device="cuda") < s["count"][:, None])[..., None]          # [batch, node, key]
    q = s["q"].view(B, T, Hk, H // Hk, D).float().permute(0, 2, 1, 3, 4).reshape(B, Hk, -1, D)
    x = (q @ k.transpose(-1, -2) / math.sqrt(D)).view(B, Hk, T, H // Hk, -1)
    x = x.masked_fill(~sees[:, None, :, None], -math.inf)
    w = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-1e30))
    total = w.sum(-1, keepdim=True)
    o = (w.view(B, Hk, -1, k.shape[2]) @ v).view(B, Hk, T, H // Hk, D) / torch.where(total > 0, total, 1)
    return o.permute(0, 2, 1, 3, 4).reshape(B, T, H * D).bfloat16()


def _own_verify(s):
    from prometorch_b200.ops.verify import verify_drafts
    return verify_drafts(s["logits"], s["tokens"], s["u"], s["temperature"], parents=s["parents"], nodes=s["count"], draft_probs=s["probs"])


def _plain_verify(s):
    B, T, V = s["logits"].shape
    node = torch.arange(T, device="cuda")
    parents = (s["parents"] if s["parents"] is not None else (node - 1).int().repeat(B, 1)).long()
    tokens, x = s["tokens"].long(), s["logits"].float()
    best = x.amax(-1, keepdim=True)
    first = torch.where(x == best, torch.arange(V, device="cuda"), V).amin(-1)              # arg-max, the lowest of equals
    t = torch.where(s["temperature"] > 0, s["temperature"], 1.0)[:, None]
    total = torch.exp((x - best) / t[..., None]).sum(-1, dtype=torch.float64)
    up = parents.clamp_min(0)
    # the weight that a node's token has at its parent, and what siblings before it with other tokens had taken
    there = torch.gather(x.gather(1, up[..., None].expand(B, T, V)), 2, tokens[..., None]).squeeze(-1).double()
    w = torch.exp((there - best.squeeze(-1).gather(1, up)) / t.double())
    real = (node < s["count"][:, None]) & (parents >= 0)
    older = (parents[:, None, :] == parents[:, :, None]) & (node[None, :] < node[:, None]) & real[:, None, :] & real[:, :, None]
    again = (older & (tokens[:, None, :] == tokens[:, :, None])).any(-1)                    # the same token a second time: nothing is left of it
    w = torch.where(again, 0, w)
    left = total.gather(1, up) - (older * w[:, None, :]).sum(-1)
    if s["probs"] is not None:
        left = left * torch.gather(s["probs"].gather(1, up[..., None].expand(B, T, V)), 2, tokens[..., None]).squeeze(-1).double()
    greedy = (s["temperature"] <= 0)[:, None]
    taken = real & torch.where(greedy, tokens == first.gather(1, up), s["u"].double() * left < w)
    chosen = taken & ~(older & taken[:, None, :]).any(-1)                                   # a parent's first child that is taken
    on = ((_sees(parents) & ~chosen[:, None, :] & (parents[:, None, :] >= 0)).sum(-1) == 0) & (node < s["count"][:, None])
    n = on.sum(1)                                                                           # nodes on the path, the first among them
    order = torch.argsort((~on).int(), dim=1, stable=True)
    path = torch.where(node < n[:, None], order, -1)
    end = order.gather(1, (n - 1).clamp_min(0)[:, None])
    # the last token: from what the rejected ones leave of the distribution at the end of the path
    y = x.gather(1, end[..., None].expand(B, 1, V)).squeeze(1).double()
    p = torch.exp((y - y.amax(-1, keepdim=True)) / t.double())
    gone = torch.zeros(B, V, device="cuda").scatter_add_(1, tokens, ((parents == end) & real).float()) > 0
    if s["probs"] is not None:
        p = p / p.sum(-1, keepdim=True)
        q = s["probs"].gather(1, end[..., None].expand(B, 1, V)).squeeze(1).double()
        p = torch.where(gone.any(-1, keepdim=True), (p - q).clamp_min(0), p)                # a whole chain was accepted: nothing is taken off
    else:
        p = torch.where(gone, 0, p)
    c = p.cumsum(-1)
    drawn = (c <= s["u"][:, :1].double() * c[:, -1:]).sum(-1)
    drawn = torch.where(greedy.squeeze(1) | (c[:, -1] <= 0), first.gather(1, end).squeeze(1), drawn)          # nothing is left: the arg-max
    out = torch.where(node < n[:, None] - 1, tokens.gather(1, torch.roll(order, -1, 1)), -1)
    out = torch.where(node == n[:, None] - 1, drawn[:, None], out)
    return path.int(), (n - 1).int(), out.int()


def _own_keep(s):
    from prometorch_b200.ops.paged_tree import paged_keep
    paged_keep(s["layers"], s["lens"], s["path"], s["count"], s["table"])
    return [s["k"], s["v"], s["ke"], s["ve"]]


def _move(t, src, old, dst, new):
    t[:, dst, :, new % PAGE] = t[:, src, :, old % PAGE]


def _plain_keep(s):
    b, j = torch.nonzero(s["path"] >= 0, as_tuple=True)
    old, new = (s["lens"].long()[b] + x for x in (s["path"].long()[b, j], j))
    src, dst = (s["table"][b, x // PAGE].long() for x in (old, new))
    [_move(t.view(torch.uint8) if t.dtype == E4M3 else t, src, old, dst, new) for t in (s["k"], s["v"], s["ke"], s["ve"]) if t is not None]
    return [s["k"], s["v"], s["ke"], s["ve"]]


# ---------------------------------------------------------------------------------------------------------------- floors
def work(case):
    """Each value that has to be read or written, once."""
    size = 1 if case.get("kind") == "e4m3" else 2
    if case["op"] == "write":
        n, H, Hk, D = case["n"], case["heads"], case["kv_heads"], case["head_dim"]
        row = 2 * (H + 2 * Hk) * D + 2 * H * D + 2 * Hk * D * size + (2 * Hk if size == 1 else 0) + (2 * Hk * D if case["want_k"] else 0) + 12
        return {"bytes": n * row, "flops": 3 * n * (H + Hk) * D}
    if case["op"] == "attend":
        B, T, H, Hk, D = case["batch"], case["nodes"], case["heads"], case["kv_heads"], case["head_dim"]
        tokens = (case["longest"] if B == 1 else case["longest"] + (B - 1) * 0.75 * case["longest"]) + 0.75 * B * T          # as prepare() draws them, on average
        return {"bytes": tokens * Hk * (2 * D * size + (2 if size == 1 else 0)) + 4 * B * T * H * D, "flops": 4 * H * D * 0.75 * T * tokens if B > 1 else 4 * H * D * T * tokens}
    if case["op"] == "verify":
        B, T, V = case["batch"], case["nodes"], case["vocab"]
        rows = B * (T if B == 1 else 1 + 0.75 * (T - 1))
        # the draft's probabilities are looked up at single tokens, but for the row that a last token is drawn from
        return {"bytes": rows * V * (2 if case["dtype"] == "bf16" else 4) + (B * V * 4 if case["drafted"] else 0), "flops": 4 * rows * V}
    moved = 0.6 * case["batch"] * (case["nodes"] - 1) + 1
    return {"bytes": 2 * case["layers"] * moved * case["kv_heads"] * (2 * case["head_dim"] * size + (2 if size == 1 else 0)), "flops": 0}


# ---------------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """The definitions in fp64, one token or request after another.  ``verify`` gives whole numbers and ``keep`` copies: nothing to compute."""
    if case["op"] in ("verify", "keep"):
        return None
    s = prepare(case, seed)
    H, Hk, D = s["heads"], s["kv_heads"], s["head_dim"]
    if case["op"] == "write":
        n = s["n"]
        x = s["qkv"].double().view(n, H + 2 * Hk, D)
        z = torch.complex(x[:, :H + Hk, :D // 2], x[:, :H + Hk, D // 2:])
        z = z * torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()][:, None]
        turned = torch.cat([z.real, z.imag], -1)
        pools = []
        for pool, exps, new in ((s["k"], s["ke"], turned[:, H:]), (s["v"], s["ve"], x[:, H + Hk:])):
            pool = pool.double()
            page, at = s["table"][s["req"].long(), s["slot"].long() // PAGE].long(), s["slot"].long() % PAGE
            if exps is not None:
                e = torch.ceil(torch.log2(new.abs().amax(-1) / LARGEST)).clamp(-64, 64)
                exps = exps.clone()
                exps[page, :, at] = (e + 127).to(torch.uint8)
                y = new / torch.exp2(e)[..., None]
                step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)     # three bits behind the first, 2^-9 the smallest step
                new = torch.round(y / step) * step
            pool[page, :, at] = new
            pools.append((pool, exps))
        (k, ke), (v, ve) = pools
        return {"q": turned[:, :H].reshape(n, H * D), "k": turned[:, H:] if s["want_k"] else None, "pages": [k, v, ke, ve]}
    B, T = s["batch"], s["nodes"]
    out = torch.zeros(B, T, H, D, dtype=torch.float64, device="cuda")
    table, lens, counts, masks = s["table"].tolist(), s["lens"].tolist(), s["count"].tolist(), s["mask"].tolist()
    for b in range(B):
        n = lens[b] + counts[b]
        pages = torch.tensor(table[b][:-(-n // PAGE)], device="cuda")
        for h in range(Hk):
            k, v = s["k"][pages, h].double().reshape(-1, D)[:n], s["v"][pages, h].double().reshape(-1, D)[:n]
            if s["ke"] is not None:
                k, v = (t * torch.exp2(e[pages, h].double().reshape(-1)[:n] - 127)[:, None] for t, e in ((k, s["ke"]), (v, s["ve"])))
            for i in range(counts[b]):
                seen = torch.tensor([j for j in range(counts[b]) if masks[b][i] >> j & 1], dtype=torch.long, device="cuda")
                kk, vv = (torch.cat([t[:lens[b]], t[lens[b] + seen]]) for t in (k, v))
                q = s["q"][b, i].double().view(H, D)[h * (H // Hk):(h + 1) * (H // Hk)]
                out[b, i, h * (H // Hk):(h + 1) * (H // Hk)] = torch.softmax(q @ kk.t() / math.sqrt(D), -1) @ vv
    return out.reshape(B, T, H * D)
