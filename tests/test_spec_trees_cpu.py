"""The batching engine with trees of drafted ids and with quantised pages, on the CPU: the same tokens in fewer passes."""
import pytest
import torch

from prometorch_b200.serve.llm import GenerationConfig, LlamaConfig, LlamaWeights, LLMEngine, Request

GREEDY = dict(temperature=0.0, repetition_penalty=1.0, top_k=1)


def tiny(**kw):
    d = dict(vocab_size=97, hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, max_position_embeddings=256, eos_token_id=-1)
    d.update(kw)
    return LlamaConfig(**d)


def prompts():
    g = torch.Generator().manual_seed(5)
    base = torch.randint(3, 97, (12,), generator=g).tolist()
    return [[1] + base * 4, [1] + torch.randint(3, 97, (20,), generator=g).tolist(), [1] + base[:5] * 9 + base[3:9] + base[:3]]


def serve(w, configs, **kw):
    eng = LLMEngine(device="cpu", max_pages=32, max_active=4, seed=3, **kw)
    eng.set_weights(w)
    for i, (p, c) in enumerate(zip(prompts(), configs)):
        eng.submit_request(Request(i, p, GenerationConfig(**c)))
    got = {}
    while eng.num_active():
        eng.step()
        got.update({r.request_id: r.token_ids for r in eng.poll_responses()})
    assert eng.kv.pages_in_use == 0
    return got, eng


@pytest.mark.parametrize("kv", [None, "e4m3"])
@pytest.mark.parametrize("branches", [1, 2, 3])
def test_trees_give_the_same_greedy_tokens(kv, branches):
    w = LlamaWeights.random(tiny(), seed=17)
    c = [dict(max_new_tokens=40, **GREEDY)] * 3
    want, plain = serve(w, c, kv_dtype=kv)
    got, tree = serve(w, c, kv_dtype=kv, spec_tokens=6, spec_branches=branches)
    assert got == want
    assert tree.spec_accepted > 0 and tree.steps < plain.steps


def test_requests_that_speculate_beside_those_that_do_not():
    """Greedy, sampled from everything, sampled from a few, with a penalty: lengths and stops hold, and a greedy neighbour's tokens stay what they were."""
    w = LlamaWeights.random(tiny(), seed=2)
    c = [dict(max_new_tokens=30, **GREEDY), dict(max_new_tokens=25, temperature=1.0, repetition_penalty=1.0, top_k=0, top_p=1.0), dict(max_new_tokens=21, temperature=0.7, repetition_penalty=1.0, top_k=5, top_p=0.9)]
    want, _ = serve(w, c)
    got, eng = serve(w, c, spec_tokens=5, spec_branches=2)
    assert got[0] == want[0] and [len(got[i]) for i in range(3)] == [30, 25, 21]
    c[1] = dict(max_new_tokens=12)                       # a penalty: one id a pass
    got, _ = serve(w, c, spec_tokens=5, spec_branches=3)
    assert got[0] == want[0] and len(got[1]) == 12
    stop = want[0][7]
    c[0] = dict(max_new_tokens=30, stop_tokens=[stop], **GREEDY)
    got, _ = serve(w, c, spec_tokens=5, spec_branches=3)
    assert got[0] == want[0][:want[0].index(stop) + 1]


def test_a_sampled_request_from_one_token_is_greedy():
    """top_k 1 at any temperature leaves one token: the tree walk draws what the arg-max gives."""
    w = LlamaWeights.random(tiny(), seed=9)
    want, _ = serve(w, [dict(max_new_tokens=24, **GREEDY)] * 3)
    got, eng = serve(w, [dict(max_new_tokens=24, temperature=0.9, top_k=1, repetition_penalty=1.0)] * 3, spec_tokens=4, spec_branches=3)
    assert got == want and eng.spec_accepted > 0


def test_quantised_pages_stay_close_to_plain_ones():
    """Logits over e4m3 pages: every cached value is off by at most 2^-4, the sums by far less."""
    w = LlamaWeights.random(tiny(), seed=4)
    ids = prompts()[0]
    rows = []
    for kv in (None, "e4m3"):
        eng = LLMEngine(device="cpu", max_pages=8, max_active=1, kv_dtype=kv)
        eng.set_weights(w)
        s = eng.open_sequence()
        eng.feed([(s, ids, [])])
        rows.append(eng.feed([(s, [5], [0])]))
        eng.close_sequence(s)
    a, b = rows
    assert not torch.equal(a, b) and float((a - b).norm() / a.norm()) < 2 ** -4


def test_the_draft_is_a_trie():
    eng = LLMEngine(device="cpu", max_pages=8, max_active=1, spec_tokens=6, spec_branches=3)
    eng.set_weights(LlamaWeights.random(tiny(), seed=1))
    hist = [7, 1, 2, 3, 4, 5, 9, 2, 3, 4, 6, 8, 3, 50, 51, 52, 1, 2, 3]
    eng.submit_request(Request(0, hist, GenerationConfig(max_new_tokens=9, **GREEDY)))
    s = eng.active[0]
    s.prompt_ids = hist
    # after 1 2 3: 4 5 9 ...; after 2 3: 4 6 8 ...; after 3: 50 51 52 ...
    ids, parents = eng._draft_tree(s, 6)
    assert ids == [4, 50, 5, 6, 51, 9] and parents == [0, 0, 1, 1, 2, 3]


def test_refusals():
    for kw in (dict(kv_dtype="int3"), dict(spec_branches=1), dict(spec_branches=4, spec_tokens=4), dict(spec_branches=1, spec_tokens=64)):
        with pytest.raises(ValueError):
            LLMEngine(device="cpu", **kw)
    from prometorch_b200.models.kifusun import KifusunConfig          # a model that has neither
    for kw in (dict(kv_dtype="e4m3"), dict(spec_tokens=2, spec_branches=1)):
        eng = LLMEngine(device="cpu", **kw)
        with pytest.raises(ValueError):
            eng.set_weights(type("W", (), {"cfg": KifusunConfig(vocab_size=64, hidden_size=32, embed_scale=1.0, eps=1e-6)})())


@pytest.mark.parametrize("kw", [dict(kv_dtype="e4m3"), dict(spec_tokens=2, spec_branches=1), dict()])
def test_more_requests_than_the_attention_of_trees_takes(kw):
    eng = LLMEngine(device="cpu", max_active=1025, max_pages=4, **kw)
    if kw:
        with pytest.raises(ValueError, match="max_active"):
            eng.set_weights(LlamaWeights.random(tiny(), seed=1))
    else:
        eng.set_weights(LlamaWeights.random(tiny(), seed=1))


def test_drafted_rows_beyond_one_launch():
    """Quantised pages, drafted ids as rows of the batch: 210 requests with four each are 1050 rows."""
    w = LlamaWeights.random(tiny(num_hidden_layers=1, hidden_size=32, num_attention_heads=2, num_key_value_heads=1), seed=6)
    got = []
    for spec in (0, 4):
        eng = LLMEngine(device="cpu", max_pages=220, max_active=210, kv_dtype="e4m3", spec_tokens=spec)
        eng.set_weights(w)
        for i in range(210):
            eng.submit_request(Request(i, [1 + i % 90, 5, 6, 7, 8, 9] * 2 + [1 + i % 90], GenerationConfig(max_new_tokens=8, **GREEDY)))
        rows = []
        forward = eng._forward_rows
        eng._draft = lambda s, k: [5, 6, 7, 8][:k]       # a draft for everybody, whatever was said before
        eng._forward_rows = lambda r, **kw: (rows.append(len(r)), forward(r, **kw))[1]
        for _ in range(3):
            eng.step()
        got.append([s.output_ids[:3] for s in eng.active])
        assert (max(rows) > 1024) == (spec > 0)
    assert got[0] == got[1]


def test_a_vocabulary_that_is_not_verified_is_refused_at_load():
    from prometorch_b200.ops.verify import MAX_VOCAB
    cfg = tiny(vocab_size=MAX_VOCAB + 1, hidden_size=128, num_attention_heads=2)
    eng = LLMEngine(device="cuda", max_pages=4, max_active=1, dtype=torch.bfloat16, spec_tokens=2, spec_branches=1)
    with pytest.raises(ValueError, match="verified"):
        eng.set_weights(type("W", (), {"cfg": cfg})())
