"""The batching engine with trees of drafted ids and quantised pages on the GPU: writing, attention, verification and keeping together, in graphs, as a server runs them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def setup(D, kv):
    from prometorch_b200.serve.llm import LlamaConfig, LlamaWeights
    cfg = LlamaConfig(vocab_size=1024, hidden_size=4 * D, intermediate_size=1024, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2, max_position_embeddings=512, eos_token_id=-1)
    g = torch.Generator().manual_seed(7)
    piece = torch.randint(3, 1024, (10,), generator=g).tolist()
    prompts = [[1] + piece * 6, [1] + torch.randint(3, 1024, (40,), generator=g).tolist(), [1] + piece[:4] * 20 + piece[2:8] + piece[:3]]
    return LlamaWeights.random(cfg, seed=2, dtype=torch.bfloat16), prompts


def serve(w, prompts, config, **kw):
    from prometorch_b200.serve.llm import GenerationConfig, LLMEngine, Request
    e = LLMEngine(device="cuda", max_pages=64, max_active=4, seed=1, **kw)
    e.set_weights(w)
    for i, p in enumerate(prompts):
        e.submit_request(Request(i, p, GenerationConfig(**config)))
    res = {}
    while e.num_active():
        e.step()
        res.update({r.request_id: r.token_ids for r in e.poll_responses()})
    assert e.kv.pages_in_use == 0
    return res, e


@pytest.mark.parametrize("kv", [None, "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
def test_greedy_tokens_of_trees(D, kv):
    """Every id that comes out is the arg-max of what the plain decode step says behind the ids before it, up to the noise of bf16 sums in another order: 3e-2 of a row's
    root mean square (the bound the engine's logits are held to against fp32), five of those on either of two logits."""
    from prometorch_b200.serve.llm import LLMEngine
    w, prompts = setup(D, kv)
    config = dict(max_new_tokens=40, temperature=0.0, repetition_penalty=1.0, top_k=1)
    for graphs in (True, False):
        got, eng = serve(w, prompts, config, spec_tokens=6, spec_branches=3, kv_dtype=kv, use_graphs=graphs)
        assert all(len(got[i]) == 40 for i in range(3)) and eng.spec_accepted > 0 and eng.steps <= 40          # a request that nothing is accepted for takes 40
        plain = LLMEngine(device="cuda", max_pages=64, max_active=4, kv_dtype=kv)
        plain.set_weights(w)
        for i, p in enumerate(prompts):
            s = plain.open_sequence()
            row = plain.feed([(s, p, [len(p) - 1])])[0]
            for t in got[i]:
                assert float(row.max() - row[t]) <= 2 * 5 * 3e-2 * float(row.square().mean().sqrt()), (i, t)
                row = plain.feed([(s, [t], [0])])[0]
            plain.close_sequence(s)


@pytest.mark.parametrize("kv", [None, "e4m3"])
def test_sampled_requests_speculate(kv):
    w, prompts = setup(64, kv)
    got, eng = serve(w, prompts, dict(max_new_tokens=30, temperature=0.05, repetition_penalty=1.0, top_k=3, top_p=0.9), spec_tokens=6, spec_branches=2, kv_dtype=kv)
    assert all(len(got[i]) == 30 for i in range(3)) and eng.spec_accepted > 0
    got, eng = serve(w, prompts, dict(max_new_tokens=9), spec_tokens=6, spec_branches=2, kv_dtype=kv)          # a penalty: one id a pass
    assert all(len(got[i]) == 9 for i in range(3)) and eng.spec_drafted == 0


def test_quantised_logits_against_the_cpu_engine():
    """The same passes in fp32 on the host over pages quantised the same way."""
    from prometorch_b200.serve.llm import LLMEngine
    w, prompts = setup(128, "e4m3")
    rows = []
    for dev in ("cuda", "cpu"):
        e = LLMEngine(device=dev, max_pages=16, max_active=2, kv_dtype="e4m3", dtype=torch.bfloat16 if dev == "cuda" else torch.float32)
        e.set_weights(w)
        s = e.open_sequence()
        e.feed([(s, prompts[0], [])])
        rows.append(torch.cat([e.feed([(s, [t], [0])]) for t in (5, 6, 7)]).float().cpu())
        e.close_sequence(s)
    a, b = rows
    assert float((a - b).norm() / b.norm()) < 5e-2          # 3e-2 as without quantising; a value near a tie of e4m3 may round either way, 2^-4 of few values


def test_head_sizes_without_kernels_are_refused():
    from prometorch_b200.serve.llm import LlamaConfig, LlamaWeights, LLMEngine
    cfg = LlamaConfig(vocab_size=64, hidden_size=64, intermediate_size=64, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=2, max_position_embeddings=64)
    w = LlamaWeights.random(cfg, seed=0, dtype=torch.bfloat16)
    for kw in (dict(kv_dtype="e4m3"), dict(spec_tokens=3, spec_branches=1)):
        with pytest.raises(ValueError):
            LLMEngine(device="cuda", max_pages=4, max_active=1, **kw).set_weights(w)


def test_drafted_rows_beyond_one_launch():
    """Quantised pages, drafted ids as rows of the batch: 129 requests with seven each share a graph of 2048 rows.  Tokens as above, for some of the requests."""
    from prometorch_b200.serve.llm import GenerationConfig, LLMEngine, Request
    w, prompts = setup(64, "e4m3")
    config = dict(max_new_tokens=10, temperature=0.0, repetition_penalty=1.0, top_k=1)
    e = LLMEngine(device="cuda", max_pages=400, max_active=129, kv_dtype="e4m3", spec_tokens=7)
    e.set_weights(w)
    for i in range(129):
        e.submit_request(Request(i, prompts[i % 3][i % 7:], GenerationConfig(**config)))
    got = {}
    while e.num_active():
        e.step()
        got.update({r.request_id: r.token_ids for r in e.poll_responses()})
    assert all(len(got[i]) == 10 for i in range(129)) and e.spec_accepted > 0
    plain = LLMEngine(device="cuda", max_pages=64, max_active=4, kv_dtype="e4m3")
    plain.set_weights(w)
    for i in (0, 63, 64, 127, 128):
        s = plain.open_sequence()
        p = prompts[i % 3][i % 7:]
        row = plain.feed([(s, p, [len(p) - 1])])[0]
        for t in got[i]:
            assert float(row.max() - row[t]) <= 2 * 5 * 3e-2 * float(row.square().mean().sqrt()), (i, t)
            row = plain.feed([(s, [t], [0])])[0]
        plain.close_sequence(s)


def test_the_number_of_drafted_ids_may_change():
    from prometorch_b200.serve.llm import GenerationConfig, LLMEngine
    w, prompts = setup(64, None)
    e = LLMEngine(device="cuda", max_pages=64, max_active=4, spec_tokens=6, spec_branches=2)
    e.set_weights(w)
    for n in (6, 3, 6, 9):
        e.spec_tokens = n
        assert e.generate(prompts[0], GenerationConfig(max_new_tokens=12, temperature=0.0, repetition_penalty=1.0, top_k=1)).tokens_generated == 12


def test_a_pass_over_trees_synchronises_once():
    """Nothing is copied to the GPU behind the pass: the host launches the verification while the layers run."""
    import warnings
    from prometorch_b200.serve.llm import GenerationConfig, LLMEngine, Request
    w, prompts = setup(64, None)
    e = LLMEngine(device="cuda", max_pages=64, max_active=4, spec_tokens=6, spec_branches=2)
    e.set_weights(w)
    for i, p in enumerate(prompts):
        e.submit_request(Request(i, p, GenerationConfig(max_new_tokens=60, temperature=0.5 * i, repetition_penalty=1.0, top_k=20)))
    for _ in range(3):
        e.step()
    waits = []
    for _ in range(6):                       # one in which no request starts a page
        with warnings.catch_warnings(record=True) as said:
            warnings.simplefilter("always")
            torch.cuda.set_sync_debug_mode("warn")
            try:
                e.step()
            finally:
                torch.cuda.set_sync_debug_mode("default")
        waits.append(sum("synchroniz" in str(x.message) for x in said))
    assert min(waits) == 1, waits
