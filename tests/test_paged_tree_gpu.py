"""Drafted tokens over the paged cache on the GPU: writing (plain and quantised), attention of trees, moving the accepted entries, against plain forms."""
import math

import pytest
import torch

from prometorch_b200.ops import paged as P
from prometorch_b200.ops import paged_tree as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
PAGE = P.PAGE


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def pools(g, n, Hk, D, kind, v_scale=None):
    """A pool of random keys and values: (k, v, k exponents, v exponents)."""
    k, v = (torch.randn(n, Hk, PAGE, D, device=DEV, generator=g) for _ in range(2))
    if v_scale is not None:
        v = v * v_scale
    if kind == "bf16":
        return k.bfloat16(), v.bfloat16(), None, None
    (k, ke), (v, ve) = R.quantise_rows(k), R.quantise_rows(v)
    return k, v, ke, ve


def table_for(lens, seed):
    need = [-(-n // PAGE) for n in lens]
    n = sum(need) + 2
    order = torch.randperm(n, generator=torch.Generator().manual_seed(seed)).int()
    table, at = torch.zeros(len(lens), max(need) + 1, dtype=torch.int32), 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    return table.to(DEV), n


def spoil(pool, exps, table, lens, value):
    """What lies behind a request's last token is anything at all."""
    for b, n in enumerate(lens):
        if n % PAGE:
            page = int(table[b, n // PAGE])
            if exps is None:
                pool[page, :, n % PAGE:] = value
            else:
                pool.view(torch.uint8)[page, :, n % PAGE:] = 0x7f
                exps[page, :, n % PAGE:] = 255


def oracle(q, H, Hk, D, lens, nodes, mask, table, k, v, ke, ve, scale):
    """In fp64: the attention, and the same weights on the values' magnitudes."""
    B, T = q.shape[:2]
    out, mag = (torch.zeros(B, T, H * D, dtype=torch.float64, device=DEV) for _ in range(2))
    for b in range(B):
        n, t = lens[b], nodes[b]
        if t == 0:
            continue
        ids = table[b, :-(-(n + t) // PAGE)].long()

        def flat(pool, exps):
            x = pool.view(torch.uint8)[ids].view(R.E4M3).double() if exps is not None else pool[ids].double()
            if exps is not None:
                x = x * torch.exp2(exps[ids].double() - 127)[..., None]
            return x.permute(1, 0, 2, 3).reshape(Hk, -1, D)[:, :n + t]
        kk, vv = flat(k, ke), flat(v, ve)
        sees = torch.zeros(t, n + t, dtype=torch.bool, device=DEV)
        sees[:, :n] = True
        for i in range(t):
            for j in range(t):
                sees[i, n + j] = bool(int(mask[b, i]) >> j & 1) if mask is not None else j <= i
        qq = q[b, :t, :H * D].double().view(t, Hk, H // Hk, D).permute(1, 0, 2, 3)                       # [Hk, t, G, D]
        x = torch.einsum("ktgd,knd->ktgn", qq, kk) * scale
        x = x.masked_fill(~sees[None, :, None], -math.inf)
        w = torch.nan_to_num(torch.softmax(x, -1), nan=0.0) * sees[None, :, None]
        vz = torch.where(sees.any(0)[None, :, None], vv, torch.zeros_like(vv))
        out[b, :t] = torch.einsum("ktgn,knd->tkgd", w, vz).reshape(t, H * D)
        mag[b, :t] = torch.einsum("ktgn,knd->tkgd", w, vz.abs()).reshape(t, H * D)
    return out, mag


def close(got, want, mag, kind):
    """One rounding of the result to bf16 (2^-8 of it); each weight rounded to the operands' type (2^-8 of it in bf16, 2^-11 in fp16), which moves the result by at most that
    share of the weighted magnitudes; fp32 scores (128 products of up to about 9 in all: 128 * 9 * 2^-24 < 2^-13) and exponentials (2^-21), once each in numerator and sum."""
    bound = 2 ** -8 * want.abs() + (2 ** -8 if kind == "bf16" else 2 ** -11) * mag + 2 ** -11 * mag + 1e-30
    worst = ((got.double() - want).abs() / bound).max()
    assert torch.isfinite(got).all()
    assert float(worst) <= 1.0, float(worst)


def random_masks(g, B, T):
    """Any bits at all, and rows without any."""
    m = torch.randint(-2 ** 63, 2 ** 63 - 1, (B, T), generator=torch.Generator().manual_seed(g), dtype=torch.int64)
    m[0, 0] = 0
    if T > 3:
        m[B - 1, 3] = 0
    return m


LENS = [0, 1, 59, 63, 64, 65, 300, 1000]


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hk,T", [(2, 2, 1), (8, 2, 1), (8, 1, 2), (6, 2, 5), (2, 1, 9), (8, 2, 8), (14, 2, 7), (3, 3, 17), (8, 2, 16), (4, 2, 64), (16, 2, 33)])
def test_trees(kind, D, H, Hk, T):
    """Every tile height and more rows than one tile holds; any masks, rows that see nothing, requests without nodes, without cached tokens, around page borders."""
    g = gen(H * 1000 + T)
    nodes = [T, max(T // 2, 1), T, T, 0, T, 1, T]
    totals = [n + T for n in LENS]
    table, n_pages = table_for(totals, T)
    k, v, ke, ve = pools(g, n_pages, Hk, D, kind)
    behind = [n + t for n, t in zip(LENS, nodes)]
    spoil(k, ke, table, behind, math.nan)
    spoil(v, ve, table, behind, math.inf)
    mask = random_masks(T, len(LENS), T)
    q = torch.randn(len(LENS), T, H * D, device=DEV, generator=g).bfloat16()
    lens = torch.tensor(LENS, dtype=torch.int32, device=DEV)
    nd = torch.tensor(nodes, dtype=torch.int32, device=DEV)
    for m in (mask.to(DEV), None):
        got = R.paged_attention_tree(q, H, Hk, D, lens, table, k, v, mask=m, nodes=nd, k_exp=ke, v_exp=ve)
        want, mag = oracle(q, H, Hk, D, LENS, nodes, m, table, k, v, ke, ve, D ** -0.5)
        P.check_status(DEV)
        close(got, want, mag, kind)
        for b, t in enumerate(nodes):
            assert not got[b, t:].any()
    assert not R.paged_attention_tree(q, H, Hk, D, lens, table, k, v, mask=mask.to(DEV), nodes=nd, k_exp=ke, v_exp=ve)[0, 0].any()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 5, 8, 16, 40])
@pytest.mark.parametrize("up", [True, False])
def test_scores_that_rise_or_fall_along_the_cache(kind, D, T, up):
    """By several powers of two from block to block: references are outgrown again and again, or the first tokens outweigh all others.

    One rounding of the result and of each weight, as everywhere; a score is off by at most D fp32 roundings of its terms' magnitudes, and (e4m3) by queries rounded to 2^-18 of the row's
    largest, which both moves the weights, in numerator and sum."""
    H, Hk, have = 8, 2, 2500
    g = gen(D + T)
    table, n_pages = table_for([have + T], 3)
    k, v, ke, ve = pools(g, n_pages, Hk, D, kind)
    place = torch.zeros(n_pages, 1, PAGE, 1, device=DEV)
    at = torch.arange(have + T, device=DEV)
    place[table[0, at // PAGE].long(), 0, at % PAGE, 0] = (at.float() / (have + T) * 6 - 3) * (1 if up else -1)
    new = place * (1 + 0.1 * torch.randn(n_pages, Hk, PAGE, D, device=DEV, generator=g))
    if kind == "e4m3":
        values, exps = R.quantise_rows(new)
        k.view(torch.uint8).copy_(values.view(torch.uint8))
        ke.copy_(exps)
    else:
        k.copy_(new.bfloat16())
    q = (1 + 0.1 * torch.randn(1, T, H * D, device=DEV, generator=g)).bfloat16()
    got = R.paged_attention_tree(q, H, Hk, D, torch.tensor([have], dtype=torch.int32, device=DEV), table, k, v, k_exp=ke, v_exp=ve)
    want, mag = oracle(q, H, Hk, D, [have], [T], None, table, k, v, ke, ve, D ** -0.5)
    terms = float(q.abs().max()) * float(new.abs().max()) * 1.0625 * D * D ** -0.5         # magnitudes of a score's terms; an e4m3 key is off by 2^-4 at most
    score = D * terms * 2 ** -24 + (2 ** -18 * terms if kind == "e4m3" else 0)
    bound = 2 ** -8 * want.abs() + (2 ** -8 if kind == "bf16" else 2 ** -11) * mag + (2 ** -11 + 2 * score) * mag + 1e-30
    assert torch.isfinite(got).all()
    assert float(((got.double() - want).abs() / bound).max()) <= 1.0


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hk,T", [(8, 2, 5), (8, 2, 8), (3, 1, 7), (4, 1, 6)])
@pytest.mark.parametrize("lens", [[540], [0], [63, 64], [1, 130]])
def test_page_tables_with_room_for_little(kind, D, H, Hk, T, lens):
    """Few pages in all: 17 to 32 rows over bf16 pages are tiles of 16."""
    g = gen(T + len(lens))
    nodes = [T, T - 2][:len(lens)]
    table, n_pages = table_for([n + T for n in lens], 3)
    k, v, ke, ve = pools(g, n_pages, Hk, D, kind)
    mask = random_masks(T, len(lens), T)
    q = torch.randn(len(lens), T, H * D, device=DEV, generator=g).bfloat16()
    got = R.paged_attention_tree(q, H, Hk, D, torch.tensor(lens, dtype=torch.int32, device=DEV), table, k, v, mask=mask.to(DEV), nodes=torch.tensor(nodes, dtype=torch.int32, device=DEV), k_exp=ke,
                                 v_exp=ve)
    want, mag = oracle(q, H, Hk, D, lens, nodes, mask, table, k, v, ke, ve, D ** -0.5)
    close(got, want, mag, kind)
    for b, n in enumerate(nodes):
        assert not got[b, n:].any()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("T", [4, 8, 16, 40])
@pytest.mark.parametrize("have", [30, 3000])
@pytest.mark.parametrize("value", [math.nan, math.inf, 2.0 ** 40])
def test_a_query_that_is_no_number_or_a_large_one(kind, T, have, value):
    """It spoils its own row, whole or cut between CTAs, and no other."""
    H, Hk, D, B = 8, 2, 128, 2
    g = gen(T)
    table, n_pages = table_for([have + T] * B, 3)
    k, v, ke, ve = pools(g, n_pages, Hk, D, kind)
    q = torch.randn(B, T, H * D, device=DEV, generator=g).bfloat16()
    lens = torch.full((B,), have, dtype=torch.int32, device=DEV)
    want, mag = oracle(q, H, Hk, D, [have] * B, [T] * B, None, table, k, v, ke, ve, D ** -0.5)
    spoilt = q.clone()
    spoilt[1, 2, 3 * D + 5] = value
    got = R.paged_attention_tree(spoilt, H, Hk, D, lens, table, k, v, k_exp=ke, v_exp=ve)
    assert got[1, 2, 3 * D:4 * D].isnan().all() or math.isfinite(value)
    got[1, 2, 3 * D:4 * D] = want[1, 2, 3 * D:4 * D].bfloat16()
    close(got, want, mag, kind)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
def test_one_node_is_the_decode_step(kind, D):
    """A whole batch of single tokens, lengths one after another: every place of the last token in a page."""
    H, Hk, B = 8, 2, 200
    g = gen(D)
    have = list(range(B))
    table, n_pages = table_for([n + 1 for n in have], 3)
    k, v, ke, ve = pools(g, n_pages, Hk, D, kind)
    q = torch.randn(B, 1, H * D, device=DEV, generator=g).bfloat16()
    got = R.paged_attention_tree(q, H, Hk, D, torch.arange(B, dtype=torch.int32, device=DEV), table, k, v, k_exp=ke, v_exp=ve, scale=0.2)
    want, mag = oracle(q, H, Hk, D, have, [1] * B, None, table, k, v, ke, ve, 0.2)
    close(got, want, mag, kind)
    if kind == "bf16":
        old = P.paged_attention_decode(q[:, 0], H, Hk, D, torch.arange(1, B + 1, dtype=torch.int32, device=DEV), table, k, v, scale=0.2)
        close(got[:, 0], old.double(), mag[:, 0] * 2, kind)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hk,T", [(4, 4, 3), (8, 4, 9), (6, 3, 20), (16, 4, 40)])
def test_many_short_items(kind, D, H, Hk, T):
    """Far more (request, tile, kv head) than there are SMs, of one block or a few each: most are one CTA's own, and it has several of them."""
    B = 150
    g = gen(D + T)
    have = [(37 * b) % 300 for b in range(B)]
    nodes = [1 + (5 * b) % T for b in range(B)]
    table, n_pages = table_for([n + T for n in have], 3)
    k, v, ke, ve = pools(g, n_pages, Hk, D, kind)
    mask = random_masks(B, B, T)
    q = torch.randn(B, T, H * D, device=DEV, generator=g).bfloat16()
    got = R.paged_attention_tree(q, H, Hk, D, torch.tensor(have, dtype=torch.int32, device=DEV), table, k, v, mask=mask.to(DEV), nodes=torch.tensor(nodes, dtype=torch.int32, device=DEV), k_exp=ke,
                                 v_exp=ve)
    want, mag = oracle(q, H, Hk, D, have, nodes, mask, table, k, v, ke, ve, D ** -0.5)
    close(got, want, mag, kind)
    for b, n in enumerate(nodes):
        assert not got[b, n:].any()


@pytest.mark.parametrize("kind,D,H,Hk,T,lens", [("e4m3", 128, 8, 2, 3, [20011]), ("bf16", 64, 8, 2, 64, [9000, 40]), ("bf16", 128, 2, 1, 1, [5, 30000, 700]), ("e4m3", 64, 4, 1, 20, [64 * 150, 64 * 150 - 20])])
def test_items_cut_between_ctas(kind, D, H, Hk, T, lens):
    g = gen(T)
    table, n_pages = table_for([n + T for n in lens], 5)
    k, v, ke, ve = pools(g, n_pages, Hk, D, kind)
    q = torch.randn(len(lens), T, H * D, device=DEV, generator=g).bfloat16()
    got = R.paged_attention_tree(q, H, Hk, D, torch.tensor(lens, dtype=torch.int32, device=DEV), table, k, v, k_exp=ke, v_exp=ve)
    want, mag = oracle(q, H, Hk, D, lens, [T] * len(lens), None, table, k, v, ke, ve, D ** -0.5)
    close(got, want, mag, kind)
    again = R.paged_attention_tree(q, H, Hk, D, torch.tensor(lens, dtype=torch.int32, device=DEV), table, k, v, k_exp=ke, v_exp=ve)
    assert torch.equal(got, again)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("T,G", [(6, 1), (8, 4), (40, 8)])
def test_no_number_in_a_masked_place(kind, T, G):
    """A drafted token whose keys and values are no numbers reaches the rows that see it and no other."""
    D, Hk, len0 = 64, 2, 77
    H, bad = Hk * G, T // 2
    g = gen(T)
    table, n_pages = table_for([len0 + T], 1)
    k, v, ke, ve = pools(g, n_pages, Hk, D, kind)
    q = torch.randn(1, T, H * D, device=DEV, generator=g).bfloat16()
    at = len0 + bad
    page = int(table[0, at // PAGE])
    for pool, value in ((k, math.nan), (v, math.inf)):
        if kind == "bf16":
            pool[page, :, at % PAGE] = value
        else:
            pool.view(torch.uint8)[page, :, at % PAGE] = 0x7f
    full = torch.tensor([[sum(1 << j for j in range(T) if j != bad)] * T], dtype=torch.int64, device=DEV)
    lens = torch.tensor([len0], dtype=torch.int32, device=DEV)
    got = R.paged_attention_tree(q, H, Hk, D, lens, table, k, v, mask=full, k_exp=ke, v_exp=ve)
    kz, vz = k.clone(), v.clone()
    for pool in (kz, vz):
        R._as_bytes(pool)[page, :, at % PAGE] = 0
    want, mag = oracle(q, H, Hk, D, [len0], [T], full, table, kz, vz, ke, ve, D ** -0.5)
    close(got, want, mag, kind)
    full[0, 1] |= 1 << bad
    got = R.paged_attention_tree(q, H, Hk, D, lens, table, k, v, mask=full, k_exp=ke, v_exp=ve)
    assert bool(torch.isnan(got[0, 1]).all())
    rest = [i for i in range(T) if i != 1]
    close(got[:, rest], want[:, rest], mag[:, rest], kind)


@pytest.mark.parametrize("T", [1, 12, 48])
def test_exponents_far_apart(T):
    """Values of very different sizes, keys that are zero, values that are zero where most of the weight lies."""
    D, H, Hk, n = 128, 4, 2, 500
    g = gen(T)
    table, n_pages = table_for([n + T], 1)
    s = torch.exp2(torch.randint(-30, 31, (n_pages, Hk, PAGE, 1), device=DEV, generator=g).float())
    k, v, ke, ve = pools(g, n_pages, Hk, D, "e4m3", v_scale=s)
    first = int(table[0, 0])
    k.view(torch.uint8)[first, :, :3], v.view(torch.uint8)[first, :, 5:9] = 0, 0
    ke[first, :, :3], ve[first, :, 5:9] = 63, 63
    q = torch.randn(1, T, H * D, device=DEV, generator=g).bfloat16() * 3
    q[0, 0, :D] = 0
    got = R.paged_attention_tree(q, H, Hk, D, torch.tensor([n], dtype=torch.int32, device=DEV), table, k, v, k_exp=ke, v_exp=ve)
    want, mag = oracle(q, H, Hk, D, [n], [T], None, table, k, v, ke, ve, D ** -0.5)
    close(got, want, mag, "bf16")           # scores three times as large: 2^-8 in place of 2^-11 covers 3 * 2^-13 with room


def test_rows_between_pieces_other_streams_and_graphs():
    D, H, Hk, T, n = 64, 4, 2, 5, 130
    g = gen(1)
    table, n_pages = table_for([n + T] * 2, 1)
    k, v, _, _ = pools(g, n_pages, Hk, D, "bf16")
    lens = torch.tensor([n, n - 9], dtype=torch.int32, device=DEV)
    wide = torch.randn(2, T, H * D + 24, device=DEV, generator=g).bfloat16()
    call = lambda q: R.paged_attention_tree(q, H, Hk, D, lens, table, k, v)  # noqa: E731
    want = call(wide[..., 8:8 + H * D].contiguous())
    for q in (wide[..., 8:], wide[..., 3:3 + H * D].contiguous()[..., :]):
        if q.shape[2] == wide.shape[2] - 8:
            assert torch.equal(call(q), want)
    odd = torch.randn(2, T, H * D + 3, device=DEV, generator=g).bfloat16()
    assert torch.equal(call(odd[..., 1:1 + H * D]), call(odd[..., 1:1 + H * D].contiguous()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(wide[..., 8:8 + H * D].contiguous())
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    # two graphs over the same operands, replayed one after the other: neither disturbs the other's workspace; lengths may change between replays
    q = wide[..., 8:8 + H * D].contiguous()
    graphs, outs = [], []
    torch.cuda.synchronize()
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(call(q))
        graphs.append(gr)
    for gr in graphs:
        gr.replay()
    assert all(torch.equal(o, want) for o in outs)
    lens.copy_(torch.tensor([3, 100], dtype=torch.int32))
    for gr in graphs:
        gr.replay()
    want = call(q)
    assert all(torch.equal(o, want) for o in outs)


def test_bad_pages_are_skipped_and_reported():
    """An id outside the pool, a length beyond the table: nothing is read there, the rest is as if those tokens were not."""
    D, H, Hk, T = 64, 2, 1, 2
    g = gen(2)
    table, n_pages = table_for([200], 1)
    k, v, _, _ = pools(g, n_pages, Hk, D, "bf16")
    q = torch.randn(1, T, H * D, device=DEV, generator=g).bfloat16()
    lens = torch.tensor([190], dtype=torch.int32, device=DEV)
    bad = table.clone()
    bad[0, 1] = n_pages
    got = R.paged_attention_tree(q, H, Hk, D, lens, bad, k, v)
    with pytest.raises(IndexError):
        P.check_status(DEV)
    kept = [0, 2, 3]
    # without the second page: the same tokens, 64 fewer in front of the drafted ones
    want, mag = oracle(q, H, Hk, D, [190 - 64], [T], None, table[:, kept].contiguous(), k, v, None, None, D ** -0.5)
    want2, mag2 = want, mag
    # the drafted tokens stand at slots 190 and 191: the last page's place is the same
    close(got, want2, mag2, "bf16")
    R.paged_attention_tree(q, H, Hk, D, torch.tensor([table.shape[1] * PAGE], dtype=torch.int32, device=DEV), table, k, v)
    with pytest.raises(IndexError):
        P.check_status(DEV)
    P.check_status(DEV)


# ---------------------------------------------------------------------------------------------- writing
def same(a, b):
    """Equal bytes, NaN codes of either sign counted as one."""
    if a.dtype == R.E4M3:
        x, y = a.float(), b.float()
        return torch.equal(torch.isnan(x), torch.isnan(y)) and torch.equal(torch.nan_to_num(x), torch.nan_to_num(y))
    return torch.equal(a, b)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("H,Hk,D", [(32, 4, 64), (32, 8, 128), (3, 3, 64), (5, 1, 128), (40, 40, 128)])
@pytest.mark.parametrize("n,slots", [(1, False), (7, True), (130, False), (515, True)])
def test_write(kind, H, Hk, D, n, slots):
    """Bit for bit what the plain form gives: rotation rounded operation by operation, one rounding to the page's type; padding rows are not stored."""
    g = gen(n + H)
    req = torch.arange(n, dtype=torch.int32) % 5
    slot = (torch.arange(n, dtype=torch.int32) // 5)
    table = torch.randperm(5 * (n // 5 // PAGE + 1), generator=torch.Generator().manual_seed(n)).int().view(5, -1)
    pos = (slot // 2 + 3) if slots else slot
    ang = torch.arange(1, n + 10, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    cos, sin = ang.cos().float(), ang.sin().float()
    if slots:
        slot[::4] = -1
    wide = torch.randn(n, (H + 2 * Hk) * D + 8, device=DEV, generator=g).bfloat16()
    pool = [torch.zeros(table.numel(), Hk, PAGE, D).bfloat16().to(R.E4M3 if kind == "e4m3" else torch.bfloat16) for _ in range(2)]
    exps = [torch.full((table.numel(), Hk, PAGE), 9, dtype=torch.uint8) if kind == "e4m3" else None for _ in range(2)]
    on = lambda t: t.to(DEV) if t is not None else None  # noqa: E731
    gpu = [on(t) for t in pool + exps]
    args = (H, Hk, D)
    for qkv in (wide, wide[:, :-8].contiguous()):
        q, k = R.paged_write(qkv, *args, on(pos), on(req), on(table), on(cos), on(sin), gpu[0], gpu[1], slot=on(slot) if slots else None, k_exp=gpu[2], v_exp=gpu[3], want_k=True)
        qc, kc = R.paged_write(qkv.cpu(), *args, pos, req, table, cos, sin, pool[0], pool[1], slot=slot if slots else None, k_exp=exps[0], v_exp=exps[1], want_k=True)
        P.check_status(DEV)
        assert torch.equal(q.cpu(), qc) and torch.equal(k.cpu(), kc)
        for a, b in zip(gpu, pool + exps):
            if a is not None:
                assert same(a.cpu(), b)


def test_write_of_values_that_are_no_numbers_and_of_any_size():
    D, H, Hk = 128, 2, 2
    rows = torch.randn(12, (H + 2 * Hk) * D, generator=torch.Generator().manual_seed(0))
    rows[0] = 0
    rows[1, ::7] = math.inf
    rows[2, 3::9] = -math.inf
    rows[3, ::5] = math.nan
    rows[4] *= 2.0 ** 100
    rows[5] *= 2.0 ** -100
    rows[6, :] = 448.0
    rows[7, :] = 449.0
    rows[8] = math.nan
    rows[9, 100:] = 0
    rows[10] *= torch.exp2(torch.arange(rows.shape[1]) % 40 - 20.0)
    rows = rows.bfloat16()
    n = rows.shape[0]
    pos = torch.zeros(n, dtype=torch.int32)
    slot, req, table = torch.arange(n, dtype=torch.int32), torch.zeros(n, dtype=torch.int32), torch.tensor([[1, 0]], dtype=torch.int32)
    cos, sin = torch.ones(1, D // 2), torch.zeros(1, D // 2)
    pool = [torch.zeros(2, Hk, PAGE, D).to(R.E4M3) for _ in range(2)]
    exps = [torch.zeros(2, Hk, PAGE, dtype=torch.uint8) for _ in range(2)]
    gpu = [t.to(DEV) for t in pool + exps]
    R.paged_write(rows.to(DEV), H, Hk, D, pos.to(DEV), req.to(DEV), table.to(DEV), cos.to(DEV), sin.to(DEV), gpu[0], gpu[1], slot=slot.to(DEV), k_exp=gpu[2], v_exp=gpu[3])
    R.paged_write(rows, H, Hk, D, pos, req, table, cos, sin, pool[0], pool[1], slot=slot, k_exp=exps[0], v_exp=exps[1])
    v = pool[1][1, :, :n].float()
    back = R.dequantise_rows(pool[1], exps[1])[1, :, :n]
    true = rows.view(n, H + 2 * Hk, D)[:, H + Hk:].transpose(0, 1).float()
    fine = torch.isfinite(true) & (true.abs() < 448 * 2.0 ** 64) & (true.abs() >= back.abs().amax(-1, keepdim=True).nan_to_num(0) * 2.0 ** -14)
    fine[:, [1, 2, 3, 8]] &= torch.isfinite(true[:, [1, 2, 3, 8]])
    assert torch.equal(torch.isnan(v), ~torch.isfinite(true))
    small = true.abs() < 2.0 ** -64
    assert bool(((back - true).abs() <= 2.0 ** -4 * true.abs())[fine & ~small].all())
    for a, b in zip(gpu, pool + exps):
        assert same(a.cpu(), b)


def test_write_reports_slots_outside():
    D, H, Hk = 64, 1, 1
    qkv = torch.randn(3, 3 * D, device=DEV).bfloat16()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    k, v, _, _ = pools(gen(0), 2, Hk, D, "bf16")
    before = k.clone()
    cos = torch.ones(4, D // 2, device=DEV)
    for pos, slot, req, table in ((i32(0, 1, 2), i32(-1, 128, -1), i32(0, 0, 0), i32(0, 1)), (i32(0, 1, 2), i32(-1, 3, -1), i32(0, 0, 0), i32(7, 1)), (i32(0, 4, 2), i32(-1, 3, -1), i32(0, 0, 0), i32(0, 1)),
                                  (i32(0, 1, 2), i32(-1, 3, -1), i32(0, 5, 0), i32(0, 1))):
        R.paged_write(qkv, H, Hk, D, pos, req, table[None], cos, torch.zeros_like(cos), k, v, slot=slot)
        with pytest.raises(IndexError):
            P.check_status(DEV)
        assert torch.equal(k, before)


# ---------------------------------------------------------------------------------------------- keeping
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("layers,B,T,Hk,D", [(1, 1, 2, 1, 64), (3, 5, 64, 2, 128), (35, 4, 19, 8, 64), (70, 2, 9, 3, 128)])
def test_keep(kind, layers, B, T, Hk, D):
    """Paths within a page and across borders, whole chains (nothing moves), requests without nodes; more layers than one launch takes."""
    lens = torch.tensor([(60 * b + 61) % 200 for b in range(B)], dtype=torch.int32)
    table, n_pages = table_for([int(n) + T for n in lens], T)
    stacks = [pools(gen(l), n_pages, Hk, D, kind) for l in range(layers)]
    h = torch.Generator().manual_seed(T)
    path, count = torch.full((B, T), -1, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        on = torch.rand(T, generator=h) < (0.5 if b != 1 else 1.1)
        on[0] = True
        ids = on.nonzero().flatten().int()
        path[b, :len(ids)], count[b] = ids, len(ids) - 1
    if B > 2:
        count[2], path[2] = -1, -1
    host = [[t.cpu() if t is not None else None for t in s] for s in stacks]
    give = (lambda s: s) if kind == "e4m3" else (lambda s: s[:2])
    R.paged_keep([give(s) for s in stacks], lens.to(DEV), path.to(DEV), count.to(DEV), table)
    R.paged_keep([give(s) for s in host], lens, path, count, table.cpu())
    P.check_status(DEV)
    for s, t in zip(stacks, host):
        for a, b in zip(s, t):
            if a is not None:
                assert torch.equal(R._as_bytes(a).cpu(), R._as_bytes(b))


def test_keep_reports_bad_pages_and_paths():
    k, v, _, _ = pools(gen(0), 3, 1, 64, "bf16")
    before = k.clone()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    for table, path in (([[0, 9]], [[0, 40]]), ([[0, 1]], [[0, 0]]), ([[0, 1]], [[0, 2]])):
        R.paged_keep([(k, v)], i32([40]), i32(path), i32([1]), i32(table))
        with pytest.raises(IndexError):
            P.check_status(DEV)
        assert torch.equal(k, before)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,G", [(6, 1), (5, 4), (8, 4), (16, 4), (20, 4), (40, 8), (64, 8)])
@pytest.mark.parametrize("cached", [False, True])
def test_a_large_token_without_weight(kind, D, T, G, cached):
    """A token 2^40 and more times as large as all others: a drafted one that nobody sees, or a cached one that half of the rows weigh with zero (and the other half with one).  What the
    others come to does not depend on it.  A score's terms are up to 2^8 (|q| to 4.5, |k| to 5, 128 of them, by D^-0.5) where the token has no weight: fp32 sums as in `close`."""
    Hk, len0 = 2, 477
    H, at = Hk * G, (300 if cached else len0 + T // 2)
    g = gen(T + D)
    table, n_pages = table_for([len0 + T], 1)
    k, v, ke, ve = pools(g, n_pages, Hk, D, kind)
    page, place = int(table[0, at // PAGE]), at % PAGE
    if kind == "bf16":
        k[page, :, place], v[page, :, place] = 2.0 ** 60, 2.0 ** 60
    else:
        for pool, exps in ((k, ke), (v, ve)):
            pool[page, :, place] = torch.full((D,), 448.0, device=DEV).to(R.E4M3)
            exps[page, :, place] = 191
    q = torch.randn(1, T, H * D, device=DEV, generator=g).bfloat16()
    full = torch.tensor([[sum(1 << j for j in range(T) if cached or len0 + j != at) - (1 << 64 if T == 64 else 0)] * T], dtype=torch.int64, device=DEV)
    lens = torch.tensor([len0], dtype=torch.int32, device=DEV)
    got = R.paged_attention_tree(q, H, Hk, D, lens, table, k, v, mask=full, k_exp=ke, v_exp=ve)
    want, mag = oracle(q, H, Hk, D, [len0], [T], full, table, k, v, ke, ve, D ** -0.5)
    small = want.abs() < 2.0 ** 30
    assert bool(small.any()) and bool((~small).any()) == cached
    close(got, want, mag, kind)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,G", [(3, 1), (8, 4), (12, 4), (20, 4), (64, 4)])
@pytest.mark.parametrize("which", [0, 1, 2, 5])
@pytest.mark.parametrize("what", [-1, -2, None, -2 ** 31, 2 ** 31 - 1])
def test_any_id_outside_the_pool(kind, D, T, G, which, what):
    """First or second page of a block, the one of the drafted tokens: reported, and the rest is as if its tokens were not there, whatever the pool's first page holds."""
    Hk, have = 2, 320
    H = Hk * G
    g = gen(T + which)
    n_pages = 9
    k, v, ke, ve = pools(g, n_pages, Hk, D, kind)
    for pool in (k, v):
        if kind == "bf16":
            pool[0] = math.nan
        else:
            pool.view(torch.uint8)[0] = 0x7f
    table = torch.tensor([[4, 2, 7, 1, 8, 3, 5]], dtype=torch.int32, device=DEV)
    bad = table.clone()
    bad[0, which] = n_pages if what is None else what
    q = torch.randn(1, T, H * D, device=DEV, generator=g).bfloat16()
    lens = torch.tensor([have], dtype=torch.int32, device=DEV)
    got = R.paged_attention_tree(q, H, Hk, D, lens, bad, k, v, k_exp=ke, v_exp=ve)
    with pytest.raises(IndexError):
        P.check_status(DEV)
    P.check_status(DEV)
    if which == 5:
        want, mag = oracle(q, H, Hk, D, [have], [T], torch.zeros(1, T, dtype=torch.int64), table, k, v, ke, ve, D ** -0.5)
    else:
        kept = [i for i in range(table.shape[1]) if i != which]
        want, mag = oracle(q, H, Hk, D, [have - PAGE], [T], None, table[:, kept].contiguous(), k, v, ke, ve, D ** -0.5)
    close(got, want, mag, kind)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_padding_may_have_any_position(kind):
    """Rows that are not stored report nothing, and q and k are what the form for the CPU gives; a stored one outside the tables is reported."""
    D, H, Hk, n = 128, 3, 2, 9
    k, v, ke, ve = pools(gen(1), 2, Hk, D, kind)
    before = R._as_bytes(k).clone()
    qkv = torch.randn(n, (H + 2 * Hk) * D, device=DEV, generator=gen(2)).bfloat16()
    ang = torch.rand(5, D // 2, generator=torch.Generator().manual_seed(1)) * 3
    cos, sin = ang.cos(), ang.sin()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    on = lambda t: t.to(DEV) if t is not None else None  # noqa: E731
    for pos, slot in ((i32(*[-1] * n), None), (i32(-5, 3, 5, 99, 4, -1, 0, 2 ** 31 - 1, -2 ** 31), i32(*[-1] * n)), (i32(-1, 2, 5, 99, 4, -1, 0, 1, -2), i32(-1, 70, -1, -1, 3, -9, 9, 127, -1))):
        args = [torch.zeros(n, dtype=torch.int32), i32(0, 1)[None], cos, sin]
        q, kk = R.paged_write(qkv, H, Hk, D, on(pos), *map(on, args), k, v, slot=on(slot), k_exp=ke, v_exp=ve, want_k=True)
        P.check_status(DEV)
        host = [t.cpu() if t is not None else None for t in (k, v, ke, ve)]
        qc, kc = R.paged_write(qkv.cpu(), H, Hk, D, pos, *args, host[0], host[1], slot=slot, k_exp=host[2], v_exp=host[3], want_k=True)
        assert torch.equal(q.cpu(), qc) and torch.equal(kk.cpu(), kc)
        assert torch.equal(R._as_bytes(k).cpu(), R._as_bytes(host[0]))
        if slot is None or int(slot.max()) < 0:
            assert torch.equal(R._as_bytes(k), before)
    R.paged_write(qkv, H, Hk, D, on(i32(*[-1] * n)), *map(on, args), k, v, slot=on(torch.arange(n, dtype=torch.int32)), k_exp=ke, v_exp=ve)
    with pytest.raises(IndexError):
        P.check_status(DEV)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("layers", [123, 124, 125, 250])
def test_keep_of_many_layers(kind, layers):
    """Up to as many as one launch takes, and more."""
    T, Hk, D = 5, 1, 64
    stacks = [pools(gen(l), 3, Hk, D, kind) for l in range(layers)]
    lens, path, count, table = (torch.tensor(x, dtype=torch.int32) for x in ([62], [[0, 2, 4, -1, -1]], [2], [[2, 0]]))
    host = [[t.cpu() if t is not None else None for t in s] for s in stacks]
    give = (lambda s: s) if kind == "e4m3" else (lambda s: s[:2])
    R.paged_keep([give(s) for s in stacks], *(t.to(DEV) for t in (lens, path, count, table)))
    R.paged_keep([give(s) for s in host], lens, path, count, table)
    P.check_status(DEV)
    for s, t in zip(stacks, host):
        for a, b in zip(s, t):
            if a is not None:
                assert torch.equal(R._as_bytes(a).cpu(), R._as_bytes(b))


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,G", [(5, 4), (8, 4), (17, 1), (32, 1), (10, 4), (40, 3)])
@pytest.mark.parametrize("B", [37, 38, 60])
def test_strange_requests_beside_others(kind, D, T, G, B):
    """In one batch, on both sides of the number of requests that another kernel takes 17 to 32 rows from: a masked token that is no number, a masked large one, a page that is none of the pool's,
    a query that is no number, requests without nodes and without cached tokens, a page table with far more room than the requests need."""
    Hk = 2
    H = Hk * G
    g = gen(T + B)
    have = [(53 * b) % 700 for b in range(B)]
    have[5] = 200
    nodes = [T if b % 4 else max(1, T - b % 3) for b in range(B)]
    nodes[7], have[8] = 0, 0
    table, n_pages = table_for([n + T for n in have], 3)
    table = torch.cat([table, torch.zeros(B, 500, dtype=torch.int32, device=DEV)], 1).contiguous()
    k, v, ke, ve = pools(g, n_pages, Hk, D, kind)
    behind = [n + t for n, t in zip(have, nodes)]
    spoil(k, ke, table, behind, math.nan)
    spoil(v, ve, table, behind, math.inf)
    mask = random_masks(B, B, T)
    q = torch.randn(B, T, H * D, device=DEV, generator=g).bfloat16()
    clean = [t.clone() if t is not None else None for t in (k, v, ke, ve)]
    for b, number in ((3, False), (4, True)):
        mask[b] &= ~(1 << 2)
        at = have[b] + 2
        page = int(table[b, at // PAGE])
        for pool, exps in ((k, ke), (v, ve)):
            if kind == "bf16":
                pool[page, :, at % PAGE] = 2.0 ** 60 if number else math.nan
            else:
                pool.view(torch.uint8)[page, :, at % PAGE] = 0x7e if number else 0x7f
                exps[page, :, at % PAGE] = 191
    lens, nd = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (have, nodes))
    given, seen, seen_have = table.clone(), table.clone(), list(have)
    given[5, 1] = -2
    seen[5] = torch.cat([table[5, :1], table[5, 2:], table[5, :1]])
    seen_have[5] -= PAGE
    want, mag = oracle(q, H, Hk, D, seen_have, nodes, mask, seen, *clean, D ** -0.5)
    strange = q.clone()
    strange[6, 1, D + 3] = math.nan
    got = R.paged_attention_tree(strange, H, Hk, D, lens, given, k, v, mask=mask.to(DEV), nodes=nd, k_exp=ke, v_exp=ve)
    with pytest.raises(IndexError):
        P.check_status(DEV)
    if int(nodes[6]) > 1 and have[6]:
        assert bool(got[6, 1, D:2 * D].isnan().all())
    got[6, 1, D:2 * D] = want[6, 1, D:2 * D].bfloat16()
    close(got, want, mag, kind)
    for b, n in enumerate(nodes):
        assert not got[b, n:].any()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,G", [(1, 4), (8, 4), (16, 4), (40, 4)])
@pytest.mark.parametrize("size", [-40, 20, 34, 36, 37, 38, 39, 40, 41, 42, 44, 60, 100, 118])
def test_queries_of_any_size(kind, D, T, G, size):
    """Up to 2^118 times the ordinary: the token with the largest score has all the weight.  No two tokens' scores are within fp32's reach of one another (a column of keys that grows by a quarter from
    token to token, in any order, decides, against others of at most 2^-10 of it)."""
    Hk, have = 2, 30
    H = Hk * G
    g = gen(T + D)
    table, n_pages = table_for([have + T], 2)
    k, v, ke, ve = pools(g, n_pages, Hk, D, kind)
    at = torch.arange(have + T, device=DEV)
    x = torch.randn(have + T, Hk, D, device=DEV, generator=g) * 2.0 ** -10
    x[:, :, 3] = 1.25 ** at[torch.randperm(have + T, device=DEV, generator=g)].float()[:, None] * 2.0 ** -20
    R.paged_write(torch.cat([x.flatten(1), torch.randn(have + T, Hk * D, device=DEV, generator=g)], 1).bfloat16(), 0, Hk, D, at.int(), torch.zeros_like(at).int(), table, torch.ones(have + T, D // 2, device=DEV),
                  torch.zeros(have + T, D // 2, device=DEV), k, v, k_exp=ke, v_exp=ve)
    q = torch.randn(1, T, H * D, device=DEV, generator=g) * 2.0 ** -12
    q[..., 3::D] = 1.0
    q = (q * 2.0 ** size).bfloat16()
    assert torch.isfinite(q).all()
    lens = torch.tensor([have], dtype=torch.int32, device=DEV)
    got = R.paged_attention_tree(q, H, Hk, D, lens, table, k, v, k_exp=ke, v_exp=ve)
    want, mag = oracle(q, H, Hk, D, [have], [T], None, table, k, v, ke, ve, D ** -0.5)
    close(got, want, mag, kind)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,G", [(1, 4), (8, 4), (16, 4), (40, 4)])
@pytest.mark.parametrize("size,keys", [(40, 0), (112, 0), (118, 0), (100, -30), (118, -30), (60, 50)])
def test_queries_large_in_every_column(kind, D, T, G, size, keys):
    """As above with all columns alike: a score is the sum of all, D times one of them, and below 2^127."""
    Hk, have = 2, 30
    H = Hk * G
    g = gen(T + D)
    table, n_pages = table_for([have + T], 2)
    k, v, ke, ve = pools(g, n_pages, Hk, D, kind)
    at = torch.arange(have + T, device=DEV)
    x = torch.ones(have + T, Hk, D, device=DEV) * 1.25 ** -at[torch.randperm(have + T, device=DEV, generator=g)].float()[:, None, None] * 2.0 ** keys
    R.paged_write(torch.cat([x.flatten(1), torch.randn(have + T, Hk * D, device=DEV, generator=g)], 1).bfloat16(), 0, Hk, D, at.int(), torch.zeros_like(at).int(), table, torch.ones(have + T, D // 2, device=DEV),
                  torch.zeros(have + T, D // 2, device=DEV), k, v, k_exp=ke, v_exp=ve)
    q = torch.full((1, T, H * D), 2.0 ** size, device=DEV).bfloat16()
    lens = torch.tensor([have], dtype=torch.int32, device=DEV)
    got = R.paged_attention_tree(q, H, Hk, D, lens, table, k, v, k_exp=ke, v_exp=ve)
    want, mag = oracle(q, H, Hk, D, [have], [T], None, table, k, v, ke, ve, D ** -0.5)
    close(got, want, mag, kind)


@pytest.mark.parametrize("T", [1, 5, 12, 48])
@pytest.mark.parametrize("n", [500, 5000])
@pytest.mark.parametrize("where", [0, 250, -1])
def test_exponents_of_values_a_hundred_apart(T, n, where):
    """One token's values of 2^44, zeros (which have the least exponent) in whole pages and among others, values of ordinary size: the sums hold, within an item and where it is cut.  Scores of
    twelve terms' size in fp32 as in `close`, three times as large: 2^-8 in place of 2^-11 covers it."""
    D, H, Hk = 128, 4, 2
    g = gen(T + n)
    table, n_pages = table_for([n + T], 1)
    k, v, ke, ve = pools(g, n_pages, Hk, D, "e4m3")
    zero = torch.rand(n_pages, Hk, PAGE, device=DEV, generator=g) < 0.3
    zero[table[0, 3:6].long()] = True
    v.view(torch.uint8)[zero], ve[zero] = 0, 63
    at = where % n
    page = int(table[0, at // PAGE])
    v[page, :, at % PAGE] = torch.full((D,), 256.0, device=DEV).to(R.E4M3)
    ve[page, :, at % PAGE] = 127 + 36
    q = torch.randn(1, T, H * D, device=DEV, generator=g).bfloat16() * 3
    got = R.paged_attention_tree(q, H, Hk, D, torch.tensor([n], dtype=torch.int32, device=DEV), table, k, v, k_exp=ke, v_exp=ve)
    want, mag = oracle(q, H, Hk, D, [n], [T], None, table, k, v, ke, ve, D ** -0.5)
    close(got, want, mag, "bf16")


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hk,T", [(64, 1, 3), (71, 1, 5), (130, 1, 2), (192, 2, 64), (63, 1, 7), (65, 1, 1), (33, 1, 2)])
def test_large_groups(kind, D, H, Hk, T):
    """Up to hundreds of heads of a kv head: a node's heads over several tiles, tiles that begin inside a node."""
    g = gen(H + T)
    have, nodes = [0, 77, 300], [T, max(1, T - 1), T]
    table, n_pages = table_for([n + T for n in have], 3)
    k, v, ke, ve = pools(g, n_pages, Hk, D, kind)
    behind = [n + t for n, t in zip(have, nodes)]
    spoil(k, ke, table, behind, math.nan)
    spoil(v, ve, table, behind, math.inf)
    mask = random_masks(T, 3, T)
    q = torch.randn(3, T, H * D, device=DEV, generator=g).bfloat16()
    lens, nd = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (have, nodes))
    got = R.paged_attention_tree(q, H, Hk, D, lens, table, k, v, mask=mask.to(DEV), nodes=nd, k_exp=ke, v_exp=ve)
    want, mag = oracle(q, H, Hk, D, have, nodes, mask, table, k, v, ke, ve, D ** -0.5)
    close(got, want, mag, kind)
    for b, n in enumerate(nodes):
        assert not got[b, n:].any()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,G,B", [(1, 4, 64), (4, 4, 64), (5, 4, 16), (8, 4, 16), (8, 4, 64), (10, 4, 16), (16, 4, 64)])
def test_weights_over_bf16_pages_keep_sixteen_bits(D, T, G, B):
    """Up to 64 rows.  Few tokens, so that roundings do not average out: the result's own rounding (2^-8 of it), each weight off by at most 2^-16 (a bf16 part leaves 2^-8,
    and the next 2^-8 of that), and fp32 scores and exponentials as in `close`."""
    Hk = 2
    H = Hk * G
    g = gen(T * G + B)
    have = [b % 9 for b in range(B)]
    table, n_pages = table_for([n + T for n in have], 3)
    k, v, _, _ = pools(g, n_pages, Hk, D, "bf16")
    q = torch.randn(B, T, H * D, device=DEV, generator=g).bfloat16()
    got = R.paged_attention_tree(q, H, Hk, D, torch.tensor(have, dtype=torch.int32, device=DEV), table, k, v)
    want, mag = oracle(q, H, Hk, D, have, [T] * B, None, table, k, v, None, None, D ** -0.5)
    bound = 2 ** -8 * want.abs() + (2 ** -16 + 2 ** -11) * mag + 1e-30
    assert float(((got.double() - want).abs() / bound).max()) <= 1.0
