"""Several drafted tokens of a request over the paged cache, plain (bf16) or quantised (e4m3): what a speculative decoding step does around the model's products.

* :func:`paged_write`: rotary + page write with the slot apart from the position (siblings of a tree share a position), quantising on the way into e4m3 pages;
* :func:`paged_attention_tree`: attention of up to 64 drafted tokens a request (one: the plain decode step) over its cached tokens and, by a bit mask, one another;
* :func:`paged_keep`: the cache entries of the accepted tokens moved to the front of the drafted ones, in every layer.

Quantised pages are :data:`E4M3` tensors ``[page, kv_head, 64, D]`` with one byte ``[page, kv_head, 64]`` for a token's keys (and one for its values) of a head: the
values stand for ``value * 2^(byte - 127)``.  The exponent is the least with ``max |x| <= 448 * 2^e``, between -64 and 64; larger magnitudes are stored as the largest,
infinities and NaN as NaN.  Attention holds for values whose exponents lie up to 100 apart (those of zeros are -64: for values up to 2^44 beside zeros).

CUDA tensors go through csrc/paged_write.cu and csrc/paged_tree.cu; CPU tensors take the plain torch form below.  A kernel that meets a page id or a
slot outside its extent skips the access and reports it: ``ops.paged.check_status`` raises."""
from __future__ import annotations

import array
import ctypes as C
import functools
import math
import operator
from typing import Optional, Sequence, Tuple

import torch

from .. import _native as N
from .paged import PAGE, _STATUS, _status

E4M3 = torch.float8_e4m3fn
MAX_NODES, MAX_REQUESTS = 64, 1024
_LARGEST, _E_MIN, _E_MAX = 448.0, -64, 64


@N.register_decls
def _decls(L):
    vp, ci, cf, ll = C.c_void_p, C.c_int, C.c_float, C.c_longlong
    if hasattr(L, "ptb_paged_write"):
        L.ptb_paged_write.argtypes = [vp, ll, ci, ci, ci, ci, vp, vp, vp, vp, ci, ci, ci, vp, vp, ci, vp, vp, vp, vp, vp, vp, vp, vp]
        L.ptb_paged_write.restype = ci
        L.ptb_paged_keep.argtypes = [vp, ci, ci, ci, ci, ci, ci, vp, vp, vp, vp, ci, vp, vp]
        L.ptb_paged_keep.restype = ci
        L.ptb_paged_attn_tree.argtypes = [vp, ll, ll, vp, ci, ci, ci, ci, ci, vp, vp, vp, vp, ci, ci, vp, vp, vp, vp, cf, vp, vp, vp]
        L.ptb_paged_attn_tree.restype = ci
        L.ptb_paged_tree_work_floats.argtypes = [ci, ci, ci, ci, ci]
        L.ptb_paged_tree_work_floats.restype = ll


def _index(t: torch.Tensor, dev: torch.device, at: int, shape: tuple, name: str) -> None:
    """int32, contiguous, on the device (`at`: its index, -1 for the host)."""
    if t.dtype is not torch.int32 or t.shape != shape or not t.is_contiguous() or t.get_device() != at:
        raise ValueError(f"{name}: a contiguous int32 tensor {list(shape)} on {dev} is needed, not {t.dtype} {list(t.shape)} on {t.device}")


def _pools(like, at: int, Hk: int, D: int, k_pages, v_pages, k_exp, v_exp) -> bool:
    """Checks a layer's pools; whether they are quantised."""
    kind, shape = k_pages.dtype, k_pages.shape
    quant = kind is E4M3
    if kind is not v_pages.dtype or not (quant or kind is like.dtype):
        raise ValueError(f"pages: {k_pages.dtype} and {v_pages.dtype} for {like.dtype} tokens")
    if len(shape) != 4 or shape[1:] != (Hk, PAGE, D) or v_pages.shape != shape:
        raise ValueError(f"pages: [page, {Hk}, {PAGE}, {D}] is needed, not {list(shape)} and {list(v_pages.shape)}")
    if (k_exp is not None) != quant or (v_exp is not None) != quant:
        raise ValueError("pages: e4m3 pages come with exponents of keys and of values, others without")
    if not (k_pages.is_contiguous() and v_pages.is_contiguous() and k_pages.get_device() == at and v_pages.get_device() == at):
        raise ValueError(f"pages: contiguous pools on {like.device} are needed")
    if quant:
        for t in (k_exp, v_exp):
            if t.dtype is not torch.uint8 or t.shape != shape[:3] or not t.is_contiguous() or t.get_device() != at:
                raise ValueError(f"pages: exponents are contiguous uint8 [page, kv head, 64] on {like.device}")
    return quant


def _launch(at: int, entry, *args) -> int:
    """Calls an entry that launches, with the device current for its length and the current stream behind the arguments."""
    if torch.cuda.current_device() == at:
        return entry(*args, _stream(at))
    with torch.cuda.device(at):
        return entry(*args, _stream(at))


def _status_ptr(dev: torch.device, at: int) -> int:
    t = _STATUS.get(at)
    return (t if t is not None else _status(dev)).data_ptr()


_shape, _dtype = operator.attrgetter("shape"), operator.attrgetter("dtype")


def _alike(tensors: Sequence[torch.Tensor], shape: tuple, dtype: torch.dtype, index: int) -> bool:
    """Contiguous, of one shape, type and device (its index, -1 for the host).  A pass over all of them for each: models have hundreds of pools, and a check in turn costs more."""
    n = len(tensors)
    return (list(map(_shape, tensors)).count(shape) == n and list(map(_dtype, tensors)).count(dtype) == n and list(map(torch.Tensor.get_device, tensors)).count(index) == n
            and all(map(torch.Tensor.is_contiguous, tensors)))


_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else lambda index: torch.cuda.current_stream(index).cuda_stream


# ---------------------------------------------------------------------------------------------- e4m3 with an exponent a row
def quantise_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x [..., D]`` as the pages hold it: e4m3 values and biased exponents ``[...]`` (plain math)."""
    x = x.float()
    sound = torch.isfinite(x)
    m, k = torch.frexp(torch.where(sound, x, torch.zeros_like(x)).abs().amax(-1, keepdim=True))
    e = torch.where(m > 0, torch.where(m <= 0.875, k - 9, k - 8), torch.full_like(k, _E_MIN)).clamp(_E_MIN, _E_MAX)          # 448 = 0.875 * 2^9
    y = torch.ldexp(x, -e).clamp(-_LARGEST, _LARGEST)
    return torch.where(sound, y, torch.full_like(y, math.nan)).to(E4M3), (e + 127).to(torch.uint8).squeeze(-1)


def dequantise_rows(values: torch.Tensor, exps: torch.Tensor) -> torch.Tensor:
    """What e4m3 ``values [..., D]`` and biased exponents ``[...]`` stand for, in fp32."""
    return torch.ldexp(values.float(), exps.int()[..., None] - 127)


def _pages_of(table_rows: torch.Tensor, n_pages: int) -> torch.Tensor:
    """Page ids as an index; an id outside the pool raises (the CUDA kernels report it instead)."""
    ids = table_rows.long()
    if bool(((ids < 0) | (ids >= n_pages)).any()):
        raise IndexError(f"paged KV: a page id outside the pool of {n_pages}")
    return ids


def _as_bytes(t: torch.Tensor) -> torch.Tensor:
    return t.view(torch.uint8) if t.dtype == E4M3 else t


# ---------------------------------------------------------------------------------------------- writing
def paged_write(qkv: torch.Tensor, H: int, Hk: int, D: int, pos: torch.Tensor, req: torch.Tensor, page_table: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                k_pages: torch.Tensor, v_pages: torch.Tensor, slot: Optional[torch.Tensor] = None, k_exp: Optional[torch.Tensor] = None,
                v_exp: Optional[torch.Tensor] = None, want_k: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rotates q and k of the ``n`` tokens of ``qkv [n, >= (H + 2 Hk) D]`` (pairs (j, j + D/2)) to the positions ``pos`` and stores k and v at
    ``page_table[req[i], slot[i] // 64]``, place ``slot[i] % 64``.  ``slot`` None: the position.  A negative one is not stored (padding), and its q and k are turned only if its
    position is one of the tables'.  Tokens of one slot are equal (rows that fill a batch up, with one id at one position).  e4m3 pages come with
    ``k_exp`` and ``v_exp``.  Returns the rotated ``q [n, H D]`` and, if asked for, the rotated keys ``[n, Hk, D]`` as they were before quantising."""
    width, dev, home = (H + 2 * Hk) * D, qkv.device, qkv.get_device()
    if qkv.dim() != 2 or qkv.shape[1] < width or H < 0 or Hk <= 0 or D <= 0 or D % 2:
        raise ValueError(f"paged_write: rows of {width} values for {H} + 2 x {Hk} heads of {D} are needed, not {list(qkv.shape)}")
    n = qkv.shape[0]
    quant = _pools(qkv, home, Hk, D, k_pages, v_pages, k_exp, v_exp)
    _index(pos, dev, home, (n,), "paged_write: pos")
    _index(req, dev, home, (n,), "paged_write: req")
    if slot is not None:
        _index(slot, dev, home, (n,), "paged_write: slot")
    if page_table.dim() != 2:
        raise ValueError("paged_write: page_table [requests, pages]")
    _index(page_table, dev, home, page_table.shape, "paged_write: page_table")
    if not (cos.dtype == sin.dtype == torch.float32 and cos.dim() == 2 and cos.shape == sin.shape and cos.shape[1] == D // 2 and cos.is_contiguous() and sin.is_contiguous()
            and cos.get_device() == home and sin.get_device() == home):
        raise ValueError(f"paged_write: contiguous fp32 tables [positions, {D // 2}] on {dev} are needed")
    if qkv.is_cuda:
        if qkv.dtype != torch.bfloat16 or D not in (64, 128):
            raise ValueError(f"paged_write: bf16 tokens with heads of 64 or 128 are needed, not {qkv.dtype} and {D}")
        ld, one = qkv.stride()
        if one != 1 or ld % 8 or ld < width or qkv.data_ptr() % 16:      # a row starts on 16 bytes
            qkv, ld = torch.empty(n, width, dtype=qkv.dtype, device=dev).copy_(qkv[:, :width]), width
        q = torch.empty(n, H * D, dtype=torch.bfloat16, device=dev)
        k = torch.empty(n, Hk, D, dtype=torch.bfloat16, device=dev) if want_k else None
        rc = _launch(home, N.lib().ptb_paged_write, qkv.data_ptr(), ld, n, H, Hk, D, pos.data_ptr(), N.ptr(slot), req.data_ptr(), page_table.data_ptr(), page_table.shape[1],
                     page_table.shape[0], k_pages.shape[0], cos.data_ptr(), sin.data_ptr(), cos.shape[0], q.data_ptr(), N.ptr(k), k_pages.data_ptr(), v_pages.data_ptr(), N.ptr(k_exp),
                     N.ptr(v_exp), _status_ptr(dev, home))
        if rc:
            N.check(rc, "paged_write")
        return q, k
    x = qkv[:, :(H + 2 * Hk) * D].reshape(n, H + 2 * Hk, D).float()
    at = (pos if slot is None else slot).long()
    keep, turns = at >= 0, (pos >= 0) & (pos < cos.shape[0])
    if bool((keep & ~turns).any()):
        raise IndexError(f"paged KV: a position outside the tables of {cos.shape[0]}")
    c, s = (torch.where(turns[:, None], t[torch.where(turns, pos, 0).long()], torch.full((), none))[:, None] for t, none in ((cos, 1.0), (sin, 0.0)))
    a, b = x[:, :H + Hk, :D // 2], x[:, :H + Hk, D // 2:]
    turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    page, at = _pages_of(page_table[req.long()[keep], at[keep] // PAGE], k_pages.shape[0]), at[keep] % PAGE
    for pages, exps, new in ((k_pages, k_exp, turned[keep][:, H:]), (v_pages, v_exp, x[keep][:, H + Hk:])):
        if quant:
            new, e = quantise_rows(new)
            exps[page, :, at] = e
        _as_bytes(pages)[page, :, at] = _as_bytes(new) if quant else new.to(pages.dtype)
    return turned[:, :H].reshape(n, H * D).to(qkv.dtype), turned[:, H:].to(qkv.dtype) if want_k else None


# ---------------------------------------------------------------------------------------------- attention
def tree_mask(parents: torch.Tensor) -> torch.Tensor:
    """``parents [B, T]`` (a node before the node, -1 for the first) -> ``[B, T]`` int64: bit j of node i, whether i is j or has it among its ancestors.  On the
    host this is a few operations for each node; keep it there."""
    B, T = parents.shape
    if not 1 <= T <= MAX_NODES:
        raise ValueError(f"tree_mask: 1 to {MAX_NODES} nodes, not {T}")
    mask = torch.zeros(B, T, dtype=torch.int64, device=parents.device)
    p = parents.long()
    if not bool(((p < torch.arange(T, device=p.device)) & (p >= -1)).all()):
        raise ValueError("tree_mask: a parent is a node before its child, or -1")
    for i in range(T):
        bit = (1 << i) - (1 << 64 if i == 63 else 0)
        up = mask.gather(1, p[:, i:i + 1].clamp_min(0)).squeeze(1)
        mask[:, i] = torch.where(p[:, i] >= 0, up, torch.zeros_like(up)) | bit
    return mask


@functools.lru_cache(maxsize=1024)
def _work_floats(B: int, T: int, H: int, Hk: int, D: int) -> int:
    return N.lib().ptb_paged_tree_work_floats(B, T, H, Hk, D)


def paged_attention_tree(q: torch.Tensor, H: int, Hk: int, D: int, lens: torch.Tensor, page_table: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                         mask: Optional[torch.Tensor] = None, nodes: Optional[torch.Tensor] = None, k_exp: Optional[torch.Tensor] = None, v_exp: Optional[torch.Tensor] = None,
                         scale: Optional[float] = None) -> torch.Tensor:
    """``q [B, T, >= H D]``: up to 64 drafted tokens of each of up to 1024 requests (heads packed along the row), node i of request b in slot ``lens[b] + i`` of the pages
    ``page_table[b]``.  It sees the ``lens[b]`` cached tokens and the nodes j of its request whose bit j is set in ``mask[b, i]`` (int64; None: a chain, nodes 0 to i).  ``nodes [B]``: how
    many of the T are there (None: all).  Returns ``[B, T, H D]``; rows behind ``nodes[b]`` and rows that see nothing are zeros.  e4m3 pages come with ``k_exp`` and ``v_exp``."""
    if q.dim() != 3 or Hk <= 0 or H <= 0 or H % Hk or q.shape[2] < H * D:
        raise ValueError(f"paged_attention_tree: [B, T, {H} x {D}] over {Hk} kv heads, not {list(q.shape)}")
    B, T, _ = q.shape
    dev, home = q.device, q.get_device()
    if not 1 <= T <= MAX_NODES:
        raise ValueError(f"paged_attention_tree: 1 to {MAX_NODES} nodes a request, not {T}")
    if B > MAX_REQUESTS:
        raise ValueError(f"paged_attention_tree: up to {MAX_REQUESTS} requests, not {B}")
    _pools(q, home, Hk, D, k_pages, v_pages, k_exp, v_exp)
    _index(lens, dev, home, (B,), "paged_attention_tree: lens")
    if nodes is not None:
        _index(nodes, dev, home, (B,), "paged_attention_tree: nodes")
    if page_table.dim() != 2 or page_table.shape[0] != B:
        raise ValueError(f"paged_attention_tree: a row of pages for each of {B} requests, not {list(page_table.shape)}")
    _index(page_table, dev, home, page_table.shape, "paged_attention_tree: page_table")
    if mask is not None and not (mask.dtype is torch.int64 and mask.shape == (B, T) and mask.is_contiguous() and mask.get_device() == home):
        raise ValueError(f"paged_attention_tree: a contiguous int64 mask [{B}, {T}] on {dev} is needed")
    scale = float(scale) if scale is not None else 1.0 / math.sqrt(D)
    if not 1e-30 < scale < 1e30:
        raise ValueError(f"paged_attention_tree: a scale above zero is needed, not {scale}")
    if q.is_cuda:
        if q.dtype != torch.bfloat16 or D not in (64, 128):
            raise ValueError(f"paged_attention_tree: bf16 queries with heads of 64 or 128 are needed, not {q.dtype} and {D}")
        s0, s1, s2 = q.stride()
        if s2 != 1 or s1 % 8 or s0 % 8 or q.data_ptr() % 16:             # a row starts on 16 bytes
            q = torch.empty(B, T, H * D, dtype=q.dtype, device=dev).copy_(q[:, :, :H * D])
            s0, s1, s2 = q.stride()
        out = torch.empty(B, T, H * D, dtype=torch.bfloat16, device=dev)
        work = torch.empty(_work_floats(B, T, H, Hk, D), dtype=torch.float32, device=dev)
        rc = _launch(home, N.lib().ptb_paged_attn_tree, q.data_ptr(), s0, s1, out.data_ptr(), B, T, H, Hk, D, lens.data_ptr(), N.ptr(nodes), N.ptr(mask), page_table.data_ptr(),
                     page_table.shape[1], k_pages.shape[0], k_pages.data_ptr(), v_pages.data_ptr(), N.ptr(k_exp), N.ptr(v_exp), scale, work.data_ptr(), _status_ptr(dev, home))
        if rc:
            N.check(rc, "paged_attention_tree")
        return out
    return paged_attention_tree_reference(q, H, Hk, D, lens, page_table, k_pages, v_pages, mask, nodes, k_exp, v_exp, scale)


def paged_attention_tree_reference(q, H, Hk, D, lens, page_table, k_pages, v_pages, mask=None, nodes=None, k_exp=None, v_exp=None, scale=None) -> torch.Tensor:
    """Softmax attention over the gathered pages, request by request and row by row (fp32, or fp64 for fp64 queries): the CPU path."""
    B, T = q.shape[:2]
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    G = H // Hk
    out = torch.zeros(B, T, H * D, dtype=q.dtype, device=q.device)
    for b in range(B):
        t = T if nodes is None else max(0, min(int(nodes[b]), T))
        n = int(lens[b])
        if n < 0 or n + t > page_table.shape[1] * PAGE:
            raise IndexError(f"paged KV: {n} cached and {t} drafted tokens in {page_table.shape[1]} pages")
        pages = _pages_of(page_table[b, :(n + t + PAGE - 1) // PAGE], k_pages.shape[0]) if t else page_table[b, :0].long()

        def flat(pool, exps):
            x = _as_bytes(pool)[pages].view(pool.dtype)
            x = dequantise_rows(x, exps[pages]) if exps is not None else x
            return x.to(wide).permute(1, 0, 2, 3).reshape(Hk, -1, D)[:, :n + t]
        k, v = flat(k_pages, k_exp), flat(v_pages, v_exp)
        for i in range(t):
            bits = int(mask[b, i]) if mask is not None else (2 << i) - 1
            sees = list(range(n)) + [n + j for j in range(t) if bits >> j & 1]
            if not sees:
                continue
            s = torch.einsum("kgd,knd->kgn", q[b, i, :H * D].to(wide).view(Hk, G, D), k[:, sees]) * scale
            out[b, i] = torch.einsum("kgn,knd->kgd", torch.softmax(s, -1), v[:, sees]).reshape(H * D).to(q.dtype)
    return out


# ---------------------------------------------------------------------------------------------- what stays
def paged_keep(layers: Sequence[Sequence[Optional[torch.Tensor]]], lens: torch.Tensor, path: torch.Tensor, count: torch.Tensor, page_table: torch.Tensor) -> None:
    """Moves the cache entries of each request's accepted drafted tokens from slot ``lens[b] + path[b, j]`` to ``lens[b] + j`` for j = 1 .. ``count[b]``, in every layer's
    pools.  ``layers``: (k_pages, v_pages) or (k_pages, v_pages, k_exp, v_exp) of each layer, of one shape; ``path [B, T]`` and ``count [B]`` are what
    :func:`~prometorch_b200.ops.verify.verify_drafts` gives (a path ascends; a count below one moves nothing); ``page_table [B, pages]``: a row for each request."""
    n = len(layers)
    if not n:
        return
    ks, vs, kes, ves = zip(*[l if len(l) == 4 else (*l, None, None) for l in layers])
    k0 = ks[0]
    dev, home, quant = k0.device, k0.get_device(), k0.dtype is E4M3
    if k0.dim() != 4 or k0.shape[2] != PAGE:
        raise ValueError(f"paged_keep: pages [page, kv head, {PAGE}, D], not {list(k0.shape)}")
    pools, exps = ks + vs, kes + ves
    if not _alike(pools, k0.shape, k0.dtype, home):
        raise ValueError("paged_keep: layers need contiguous pools of one shape, type and device")
    there = sum(map(torch.is_tensor, exps))
    if not quant and there:
        raise ValueError("paged_keep: only e4m3 pools have exponents")
    if quant and (there != 2 * n or not _alike(exps, k0.shape[:3], torch.uint8, home)):
        raise ValueError(f"paged_keep: exponents are contiguous uint8 [page, kv head, {PAGE}] on {dev}, for e4m3 pools all of them")
    if path.dim() != 2 or page_table.dim() != 2 or page_table.shape[0] != path.shape[0]:
        raise ValueError(f"paged_keep: a path [B, T] and a row of pages for each request, not {list(path.shape)} and {list(page_table.shape)}")
    B, T = path.shape
    if T > MAX_NODES:
        raise ValueError(f"paged_keep: up to {MAX_NODES} nodes a request, not {T}")
    _index(path, dev, home, (B, T), "paged_keep: path")
    _index(lens, dev, home, (B,), "paged_keep: lens")
    _index(count, dev, home, (B,), "paged_keep: count")
    _index(page_table, dev, home, page_table.shape, "paged_keep: page_table")
    if k0.is_cuda:
        row = k0.shape[3] * k0.element_size()
        if row % 16:
            raise ValueError(f"paged_keep: rows of 16-byte pieces are needed, not {row} bytes")
        at = list(map(torch.Tensor.data_ptr, pools + exps)) if quant else list(map(torch.Tensor.data_ptr, pools)) + [0] * (2 * n)
        ptrs = array.array("Q", at)                  # all keys, all values, all exponents of keys, all of values
        rc = _launch(home, N.lib().ptb_paged_keep, ptrs.buffer_info()[0], n, B, T, k0.shape[1], row, k0.shape[0], lens.data_ptr(), path.data_ptr(), count.data_ptr(), page_table.data_ptr(),
                     page_table.shape[1], _status_ptr(dev, home))
        if rc:
            N.check(rc, "paged_keep")
        return
    flat = pools + exps
    for b in range(B):
        n = min(int(count[b]), T - 1)
        if n < 1:
            continue
        old, new = int(lens[b]) + path[b, 1:n + 1].long(), int(lens[b]) + torch.arange(1, n + 1)
        src, dst = _pages_of(page_table[b, old // PAGE], k0.shape[0]), _pages_of(page_table[b, new // PAGE], k0.shape[0])
        for t in flat:
            if t is not None:
                _as_bytes(t)[dst, :, new % PAGE] = _as_bytes(t)[src, :, old % PAGE]
