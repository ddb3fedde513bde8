"""Drafted tokens over the paged cache: the plain forms against independent ones, and what is refused (on the host, before any launch)."""
import math

import pytest
import torch

from prometorch_b200.ops import paged_tree as R
from prometorch_b200.ops.paged import PAGE, paged_attention_reference, paged_rope_write

BASE = 1 << 20          # an aligned address; nothing is read from it


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def pools(n, Hk, D, quant, seed=0):
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(n, Hk, PAGE, D, generator=g) for _ in range(2))
    if not quant:
        return k, v, None, None
    (k, ke), (v, ve) = R.quantise_rows(k), R.quantise_rows(v)
    return k, v, ke, ve


# ---------------------------------------------------------------------------------------------- plain forms
def test_quantised_rows_round_to_nearest_with_the_least_exponent():
    x = torch.randn(50, 64, generator=torch.Generator().manual_seed(1)) * torch.exp2(torch.arange(50.0) - 25)[:, None]
    q, e = R.quantise_rows(x)
    a = x.abs().amax(-1)
    s = torch.exp2(e.float() - 127)
    assert bool((a <= 448 * s).all()) and bool((a > 224 * s).all())
    codes = torch.arange(256, dtype=torch.uint8).view(R.E4M3).float()
    codes = codes[torch.isfinite(codes)]
    best = (x[..., None].double() / s[:, None, None] - codes).abs().amin(-1)
    assert torch.equal((x.double() / s[:, None] - q.double()).abs(), best)
    assert torch.equal(R.dequantise_rows(q, e), q.float() * s[:, None])


def test_quantised_rows_of_no_numbers_and_zeros():
    x = torch.zeros(5, 16)
    x[1, 3], x[2, 4], x[3, 5] = math.inf, math.nan, -math.inf
    x[1, 0] = 3.0
    x[4, :] = 2.0 ** 90
    q, e = R.quantise_rows(x)
    assert e.tolist() == [63, 127 - 7, 63, 63, 191]
    assert torch.isnan(q.float()).nonzero().tolist() == [[1, 3], [2, 4], [3, 5]]
    assert float(q[1, 0]) * 2.0 ** -7 == 3.0 and bool((q[4].float() == 448).all())


@pytest.mark.parametrize("quant", [False, True])
def test_chains_of_one_are_the_decode_step(quant):
    H, Hk, D, lens = 4, 2, 64, [0, 5, 63, 64, 130]
    table = torch.randperm(20, generator=torch.Generator().manual_seed(2)).int()[:15].view(5, 3)
    k, v, ke, ve = pools(20, Hk, D, quant)
    q = torch.randn(5, 1, H * D, generator=torch.Generator().manual_seed(3))
    got = R.paged_attention_tree(q, H, Hk, D, i32(*lens), table, k, v, k_exp=ke, v_exp=ve)
    kf, vf = (R.dequantise_rows(k, ke), R.dequantise_rows(v, ve)) if quant else (k, v)
    want = paged_attention_reference(q[:, 0], H, Hk, D, i32(*lens) + 1, table, kf, vf)
    assert torch.allclose(got[:, 0], want, atol=1e-5)


def test_a_tree_is_its_branches():
    """Every node's row is what the chain of its ancestors gives, written as a chain."""
    H, Hk, D, n = 4, 2, 64, 70
    parents = i32(-1, 0, 0, 1, 2, 2, 5)[None]
    T = parents.shape[1]
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(T, (H + 2 * Hk) * D, generator=g)
    cos, sin = torch.rand(200, D // 2, generator=g), torch.rand(200, D // 2, generator=g)
    table = i32(3, 1)[None]
    mask = R.tree_mask(parents)
    depth = [0] * T
    for i in range(1, T):
        depth[i] = depth[int(parents[0, i])] + 1
    k, v, _, _ = pools(4, Hk, D, False)
    base = k.clone(), v.clone()
    q, _ = R.paged_write(qkv, H, Hk, D, i32(*[n + d for d in depth]), i32(*[0] * T), table, cos, sin, k, v, slot=torch.arange(n, n + T, dtype=torch.int32))
    got = R.paged_attention_tree(q[None], H, Hk, D, i32(n), table, k, v, mask=mask)
    for i in range(T):
        line, at = [], i
        while at >= 0:
            line.append(at)
            at = int(parents[0, at])
        line.reverse()
        kk, vv = base[0].clone(), base[1].clone()
        rows = qkv[line].clone()
        m = len(line)
        paged_rope_write(rows, H, Hk, D, torch.arange(n, n + m, dtype=torch.int32), i32(*[0] * m), table, cos, sin, kk, vv)
        want = paged_attention_reference(rows[-1:, :H * D], H, Hk, D, i32(n + m), table, kk, vv)
        assert torch.allclose(got[0, i], want[0], atol=1e-5), i
        # once the line is accepted and its entries moved, the cache is that chain's
        k2, v2 = k.clone(), v.clone()
        R.paged_keep([(k2, v2)], i32(n), i32(*(line + [-1] * (T - m)))[None], i32(m - 1), table)
        for a, b in ((k2, kk), (v2, vv)):
            flat = lambda t: t[table[0].long()].permute(0, 2, 1, 3).reshape(2 * PAGE, Hk, D)[:n + m]  # noqa: E731
            assert torch.allclose(flat(a), flat(b), atol=1e-6)


def test_tree_mask():
    m = R.tree_mask(torch.arange(-1, 63, dtype=torch.int32)[None])[0]
    assert int(m[0]) == 1 and int(m[5]) == 63 and int(m[63]) == -1 and int(m[62]) == 2 ** 63 - 1
    assert R.tree_mask(i32(-1, 0, 0, 1)[None]).tolist() == [[1, 3, 5, 11]]
    with pytest.raises(ValueError):
        R.tree_mask(i32(-1, 1)[None])
    with pytest.raises(ValueError):
        R.tree_mask(torch.zeros(1, 65, dtype=torch.int32))


def test_rows_that_see_nothing_and_requests_without_nodes():
    k, v, _, _ = pools(2, 1, 64, False)
    q = torch.randn(2, 3, 64)
    got = R.paged_attention_tree(q, 1, 1, 64, i32(0, 0), i32(0, 1).view(2, 1), k, v, mask=torch.tensor([[0, 3, 4], [1, 1, 1]]), nodes=i32(3, 0))
    assert not got[0, 0].any() and got[0, 1].any() and not got[1].any()


# ---------------------------------------------------------------------------------------------- refusals
def call_attend(**kw):
    k, v, ke, ve = pools(2, 2, 64, kw.pop("quant", False))
    a = dict(q=torch.randn(1, 3, 4 * 64), H=4, Hk=2, D=64, lens=i32(5), page_table=i32(0, 1)[None], k_pages=k, v_pages=v, k_exp=ke, v_exp=ve)
    a.update(kw)
    return R.paged_attention_tree(**a)


@pytest.mark.parametrize("kw", [dict(H=3), dict(Hk=0), dict(q=torch.randn(1, 65, 256)), dict(q=torch.randn(1, 3, 255)), dict(q=torch.randn(3, 256)), dict(lens=torch.tensor([5])), dict(lens=i32(5, 5)),
                                dict(page_table=i32(0, 1)), dict(page_table=i32(0, 1, 0, 1).view(2, 2)), dict(nodes=i32(1, 1)), dict(mask=torch.zeros(1, 3, dtype=torch.int32)),
                                dict(mask=torch.zeros(1, 2, dtype=torch.int64)), dict(k_exp=torch.zeros(2, 2, 64, dtype=torch.uint8)), dict(k_pages=torch.zeros(2, 2, 64, 32)),
                                dict(v_pages=torch.zeros(3, 2, 64, 64)), dict(quant=True, k_exp=None), dict(quant=True, v_exp=torch.zeros(2, 2, 64)), dict(k_pages=torch.zeros(2, 2, 64, 64).bfloat16()),
                                dict(k_pages=torch.zeros(2, 64, 2, 64).transpose(1, 2)), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf)])
def test_attention_refuses(kw):
    with pytest.raises(ValueError):
        call_attend(**kw)


def test_attention_refuses_more_requests_than_a_launch_can_plan():
    n = R.MAX_REQUESTS + 1
    with pytest.raises(ValueError, match="requests"):
        call_attend(q=torch.zeros(n, 1, 256), lens=torch.zeros(n, dtype=torch.int32), page_table=torch.zeros(n, 1, dtype=torch.int32))


@pytest.mark.parametrize("kw", [dict(page_table=i32(0, 2)[None], lens=i32(70)), dict(page_table=i32(-1, 0)[None]), dict(lens=i32(126)), dict(lens=i32(-1))])
def test_attention_outside_the_pool(kw):
    with pytest.raises(IndexError):
        call_attend(**kw)


def call_write(**kw):
    k, v, ke, ve = pools(2, 2, 64, kw.pop("quant", False))
    a = dict(qkv=torch.randn(3, 8 * 64), H=4, Hk=2, D=64, pos=i32(0, 1, 2), req=i32(0, 0, 0), page_table=i32(0, 1)[None], cos=torch.zeros(9, 32), sin=torch.zeros(9, 32), k_pages=k, v_pages=v, k_exp=ke,
             v_exp=ve)
    a.update(kw)
    return R.paged_write(**a)


@pytest.mark.parametrize("kw", [dict(qkv=torch.randn(3, 8 * 64 - 1)), dict(qkv=torch.randn(2, 8 * 64)), dict(pos=torch.arange(3)), dict(slot=i32(1, 2)), dict(req=i32(0)), dict(cos=torch.zeros(9, 64)),
                                dict(sin=torch.zeros(9, 32).double()), dict(page_table=i32(0, 1)), dict(quant=True, v_exp=None), dict(k_exp=torch.zeros(2, 2, 64, dtype=torch.uint8)), dict(D=32),
                                dict(v_pages=torch.zeros(2, 2, 64, 64).to(R.E4M3))])
def test_write_refuses(kw):
    with pytest.raises(ValueError):
        call_write(**kw)


def test_write_outside_the_pool():
    with pytest.raises(IndexError):
        call_write(page_table=i32(5, 1)[None])


def test_keep_refuses():
    k, v, _, _ = pools(2, 1, 64, False)
    q, w, ke, ve = pools(2, 1, 64, True)
    ok = dict(lens=i32(3), path=i32(0, 2)[None], count=i32(1), page_table=i32(0, 1)[None])
    R.paged_keep([], **ok)
    for layers in ([(k, v[:1])], [(k, v), (k.bfloat16(), v.bfloat16())], [(k, v, ke, ve)], [(q, w)], [(q, w, ke, ve.float())], [(k.transpose(2, 3).contiguous().transpose(2, 3), v)]):
        with pytest.raises(ValueError):
            R.paged_keep(layers, **ok)
    for bad in (dict(lens=i32(3, 3)), dict(path=i32(0, 2)), dict(count=torch.tensor([1])), dict(page_table=i32(0, 1))):
        with pytest.raises(ValueError):
            R.paged_keep([(k, v)], **{**ok, **bad})
    with pytest.raises(IndexError):
        R.paged_keep([(k, v)], **{**ok, "page_table": i32(7, 1)[None]})


def refused(rc):
    from prometorch_b200 import _native as N
    return rc == -1 and N.lib().ptb_last_error().decode()


def test_native_entries_refuse():
    """Operands that a kernel could not read, from a C caller."""
    import ctypes as C
    from prometorch_b200 import _native as N
    L = N.lib()

    def attend(q=BASE, q_batch=1024, q_row=512, B=1, T=2, H=4, Hk=2, D=128, stride=4, pages=8, k=BASE, v=BASE, ke=None, ve=None, work=BASE):
        return refused(L.ptb_paged_attn_tree(q, q_batch, q_row, BASE, B, T, H, Hk, D, BASE, None, None, BASE, stride, pages, k, v, ke, ve, 1.0, work, BASE, None))
    for kw, word in ((dict(T=65), "nodes"), (dict(T=0), "nodes"), (dict(B=5000), "requests"), (dict(H=5), "heads"), (dict(D=96), "head size"), (dict(q=BASE + 8), "16 bytes"), (dict(q_row=516), "16 bytes"),
                     (dict(k=BASE + 8), "16-byte"), (dict(v=BASE + 4), "16-byte"), (dict(ke=BASE), "belong together"), (dict(work=BASE + 8), "16-byte"), (dict(stride=0), "no pages"),
                     (dict(pages=1 << 28), "31 bits")):
        assert word in (attend(**kw) or ""), kw

    def write(qkv=BASE, ld=1024, D=128, k=BASE, ke=None, ve=None, cos=BASE):
        return refused(L.ptb_paged_write(qkv, ld, 3, 4, 2, D, BASE, None, BASE, BASE, 2, 1, 8, cos, BASE, 9, BASE, None, k, BASE, ke, ve, BASE, None))
    for kw, word in ((dict(D=80), "head size"), (dict(ld=1020), "multiple of eight"), (dict(ld=512), "multiple of eight"), (dict(qkv=BASE + 2), "aligned"), (dict(k=BASE + 8), "aligned"),
                     (dict(cos=BASE + 4), "aligned"), (dict(ve=BASE), "belong together")):
        assert word in (write(**kw) or ""), kw
    ptrs = (C.c_void_p * 4)(BASE, BASE + 8, None, None)
    assert "aligned" in (refused(L.ptb_paged_keep(ptrs, 1, 1, 4, 2, 128, 8, BASE, BASE, BASE, BASE, 4, BASE, None)) or "")
    ptrs = (C.c_void_p * 4)(BASE, BASE, BASE, None)
    assert "exponents" in (refused(L.ptb_paged_keep(ptrs, 1, 1, 4, 2, 128, 8, BASE, BASE, BASE, BASE, 4, BASE, None)) or "")
    assert "bytes" in (refused(L.ptb_paged_keep(ptrs, 1, 1, 4, 2, 100, 8, BASE, BASE, BASE, BASE, 4, BASE, None)) or "")
    assert L.ptb_paged_write(BASE, 1024, 0, 4, 2, 128, BASE, None, BASE, BASE, 2, 1, 8, BASE, BASE, 9, BASE, None, BASE, BASE, None, None, BASE, None) == 0


def test_padding_may_have_any_position():
    """Rows that are not stored: q and k are turned where the tables reach, else left as they are; a stored row outside the tables raises."""
    D, H, Hk = 64, 2, 1
    k, v, _, _ = pools(2, Hk, D, False)
    before = k.clone()
    qkv = torch.randn(4, (H + 2 * Hk) * D, generator=torch.Generator().manual_seed(1))
    ang = torch.rand(5, D // 2) * 3
    call = lambda pos, slot: R.paged_write(qkv, H, Hk, D, pos, i32(0, 0, 0, 0), i32(0, 1)[None], ang.cos(), ang.sin(), k, v, slot=slot, want_k=True)  # noqa: E731
    q, kk = call(i32(-1, -7, -1, -2), None)
    assert torch.equal(q, qkv[:, :H * D]) and torch.equal(kk[:, 0], qkv[:, H * D:(H + 1) * D]) and torch.equal(k, before)
    q, _ = call(i32(3, 5, -1, 99), i32(-1, -1, -1, -1))
    assert torch.equal(q[1:], qkv[1:, :H * D]) and not torch.equal(q[0], qkv[0, :H * D]) and torch.equal(k, before)
    for pos in (i32(0, 5, 1, 2), i32(0, -1, 1, 2)):
        with pytest.raises(IndexError):
            call(pos, i32(0, 1, 2, 3))
