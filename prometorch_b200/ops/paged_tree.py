"""Several drafted tokens of a request over the paged cache, plain (bf16) or quantised (e4m3): what a speculative decoding step does around the model's products.

* :func:`paged_write`: rotary + page write with the slot apart from the position (siblings of a tree share a position), quantising on the way into e4m3 pages;
* :func:`paged_attention_tree`: attention of up to 64 drafted tokens a request (one: the plain decode step) over its cached tokens and, by a bit mask, one another;
* :func:`paged_keep`: the cache entries of the accepted tokens moved to the front of the drafted ones, in every layer.

Quantised pages are :data:`E4M3` tensors ``[page, kv_head, 64, D]`` with one byte ``[page, kv_head, 64]`` for a token's keys (and one for its values) of a head: the
values stand for ``value * 2^(byte - 127)``.  The exponent is the least with ``max |x| <= 448 * 2^e``, between -64 and 64; larger magnitudes are stored as the largest,
infinities and NaN as NaN.

CUDA tensors go through csrc/paged_write.cu and csrc/paged_tree.cu; CPU tensors take the plain torch form below.  A kernel that meets a page id or a
slot outside its extent skips the access and reports it: ``ops.paged.check_status`` raises."""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Sequence, Tuple

import torch

from .. import _native as N
from .paged import PAGE, _status

E4M3 = torch.float8_e4m3fn
MAX_NODES = 64
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
        L.ptb_paged_tree_work_floats.argtypes = [ci, ci, ci, ci]
        L.ptb_paged_tree_work_floats.restype = ll


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _index(t: torch.Tensor, like: torch.Tensor, shape: tuple, name: str) -> None:
    """int32, contiguous, on the device of ``like``."""
    if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous() or t.device != like.device:
        raise ValueError(f"{name}: a contiguous int32 tensor {list(shape)} on {like.device} is needed, not {t.dtype} {list(t.shape)} on {t.device}")


def _pools(like, Hk: int, D: int, k_pages, v_pages, k_exp, v_exp) -> bool:
    """Checks a layer's pools; whether they are quantised."""
    quant = k_pages.dtype == E4M3
    _need(k_pages.dtype == v_pages.dtype and (quant or k_pages.dtype == like.dtype), f"pages: {k_pages.dtype} and {v_pages.dtype} for {like.dtype} tokens")
    _need(k_pages.dim() == 4 and tuple(k_pages.shape[1:]) == (Hk, PAGE, D) and k_pages.shape == v_pages.shape,
          f"pages: [page, {Hk}, {PAGE}, {D}] is needed, not {list(k_pages.shape)} and {list(v_pages.shape)}")
    _need((k_exp is not None) == quant and (v_exp is not None) == quant, "pages: e4m3 pages come with exponents of keys and of values, others without")
    for t in (k_pages, v_pages) + ((k_exp, v_exp) if quant else ()):
        _need(t.is_contiguous() and t.device == like.device, f"pages: contiguous pools on {like.device} are needed")
    if quant:
        _need(k_exp.dtype == v_exp.dtype == torch.uint8 and k_exp.shape == v_exp.shape == k_pages.shape[:3], "pages: exponents are uint8 [page, kv head, 64]")
    return quant


def _on(t: torch.Tensor):
    """The current stream of the tensor's device, for a launch on it."""
    return torch.cuda.current_stream(t.device).cuda_stream


class _Device:
    """Makes a tensor's device the current one for the length of a launch, if it is not."""

    def __init__(self, t: torch.Tensor):
        self.index = t.device.index

    def __enter__(self):
        self.old = torch.cuda.current_device()
        if self.old != self.index:
            torch.cuda.set_device(self.index)

    def __exit__(self, *_):
        if self.old != self.index:
            torch.cuda.set_device(self.old)


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
    ``page_table[req[i], slot[i] // 64]``, place ``slot[i] % 64``.  ``slot`` None: the position; a negative one is not stored (padding).  No two tokens have one slot.  e4m3 pages
    come with ``k_exp`` and ``v_exp``.  Returns the rotated ``q [n, H D]`` and, if asked for, the rotated keys ``[n, Hk, D]`` as they were before quantising."""
    n = qkv.shape[0]
    _need(qkv.dim() == 2 and qkv.shape[1] >= (H + 2 * Hk) * D and H >= 0 and Hk > 0 and D > 0 and D % 2 == 0,
          f"paged_write: rows of {(H + 2 * Hk) * D} values for {H} + 2 x {Hk} heads of {D} are needed, not {list(qkv.shape)}")
    quant = _pools(qkv, Hk, D, k_pages, v_pages, k_exp, v_exp)
    for t, name in ((pos, "pos"), (req, "req")) + (((slot, "slot"),) if slot is not None else ()):
        _index(t, qkv, (n,), "paged_write: " + name)
    _need(page_table.dim() == 2, "paged_write: page_table [requests, pages]")
    _index(page_table, qkv, tuple(page_table.shape), "paged_write: page_table")
    _need(cos.dtype == sin.dtype == torch.float32 and cos.shape == sin.shape and cos.dim() == 2 and cos.shape[1] == D // 2 and cos.is_contiguous() and sin.is_contiguous()
          and cos.device == sin.device == qkv.device, f"paged_write: contiguous fp32 tables [positions, {D // 2}] on {qkv.device} are needed")
    if qkv.is_cuda:
        _need(qkv.dtype == torch.bfloat16 and D in (64, 128), f"paged_write: bf16 tokens with heads of 64 or 128 are needed, not {qkv.dtype} and {D}")
        if qkv.stride(1) != 1 or qkv.stride(0) % 8 or qkv.stride(0) < (H + 2 * Hk) * D or qkv.data_ptr() % 16:      # a row starts on 16 bytes
            qkv = qkv[:, :(H + 2 * Hk) * D].contiguous() if qkv.stride(1) != 1 or qkv.shape[1] != (H + 2 * Hk) * D else qkv.clone(memory_format=torch.contiguous_format)
        q = torch.empty(n, H * D, dtype=qkv.dtype, device=qkv.device)
        k = torch.empty(n, Hk, D, dtype=qkv.dtype, device=qkv.device) if want_k else None
        with _Device(qkv):
            N.check(N.lib().ptb_paged_write(qkv.data_ptr(), qkv.stride(0), n, H, Hk, D, pos.data_ptr(), N.ptr(slot), req.data_ptr(), page_table.data_ptr(), page_table.stride(0),
                                            page_table.shape[0], k_pages.shape[0], cos.data_ptr(), sin.data_ptr(), cos.shape[0], q.data_ptr(), N.ptr(k), k_pages.data_ptr(),
                                            v_pages.data_ptr(), N.ptr(k_exp), N.ptr(v_exp), _status(qkv.device).data_ptr(), _on(qkv)), "paged_write")
        return q, k
    x = qkv[:, :(H + 2 * Hk) * D].reshape(n, H + 2 * Hk, D).float()
    c, s = cos[pos.long()][:, None], sin[pos.long()][:, None]
    a, b = x[:, :H + Hk, :D // 2], x[:, :H + Hk, D // 2:]
    turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    at = (pos if slot is None else slot).long()
    keep = at >= 0
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
    _need(1 <= T <= MAX_NODES, f"tree_mask: 1 to {MAX_NODES} nodes, not {T}")
    mask = torch.zeros(B, T, dtype=torch.int64, device=parents.device)
    p = parents.long()
    _need(bool(((p < torch.arange(T, device=p.device)) & (p >= -1)).all()), "tree_mask: a parent is a node before its child, or -1")
    for i in range(T):
        bit = (1 << i) - (1 << 64 if i == 63 else 0)
        up = mask.gather(1, p[:, i:i + 1].clamp_min(0)).squeeze(1)
        mask[:, i] = torch.where(p[:, i] >= 0, up, torch.zeros_like(up)) | bit
    return mask


def paged_attention_tree(q: torch.Tensor, H: int, Hk: int, D: int, lens: torch.Tensor, page_table: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                         mask: Optional[torch.Tensor] = None, nodes: Optional[torch.Tensor] = None, k_exp: Optional[torch.Tensor] = None, v_exp: Optional[torch.Tensor] = None,
                         scale: Optional[float] = None) -> torch.Tensor:
    """``q [B, T, >= H D]``: up to 64 drafted tokens of each request (heads packed along the row), node i of request b in slot ``lens[b] + i`` of the pages
    ``page_table[b]``.  It sees the ``lens[b]`` cached tokens and the nodes j of its request whose bit j is set in ``mask[b, i]`` (int64; None: a chain, nodes 0 to i).  ``nodes [B]``: how
    many of the T are there (None: all).  Returns ``[B, T, H D]``; rows behind ``nodes[b]`` and rows that see nothing are zeros.  e4m3 pages come with ``k_exp`` and ``v_exp``."""
    _need(q.dim() == 3 and q.shape[2] >= H * D and Hk > 0 and H > 0 and H % Hk == 0, f"paged_attention_tree: [B, T, {H} x {D}] over {Hk} kv heads, not {list(q.shape)}")
    B, T = q.shape[:2]
    _need(1 <= T <= MAX_NODES, f"paged_attention_tree: 1 to {MAX_NODES} nodes a request, not {T}")
    quant = _pools(q, Hk, D, k_pages, v_pages, k_exp, v_exp)
    _index(lens, q, (B,), "paged_attention_tree: lens")
    if nodes is not None:
        _index(nodes, q, (B,), "paged_attention_tree: nodes")
    _need(page_table.dim() == 2 and page_table.shape[0] == B, f"paged_attention_tree: a row of pages for each of {B} requests, not {list(page_table.shape)}")
    _index(page_table, q, tuple(page_table.shape), "paged_attention_tree: page_table")
    if mask is not None:
        _need(mask.dtype == torch.int64 and tuple(mask.shape) == (B, T) and mask.is_contiguous() and mask.device == q.device,
              f"paged_attention_tree: a contiguous int64 mask [{B}, {T}] on {q.device} is needed")
    scale = float(scale) if scale is not None else 1.0 / math.sqrt(D)
    if q.is_cuda:
        _need(q.dtype == torch.bfloat16 and D in (64, 128), f"paged_attention_tree: bf16 queries with heads of 64 or 128 are needed, not {q.dtype} and {D}")
        if q.stride(2) != 1 or q.stride(1) % 8 or q.stride(0) % 8 or q.data_ptr() % 16:
            q = q.clone(memory_format=torch.contiguous_format) if (q.shape[2] % 8 == 0) else q[:, :, :H * D].clone(memory_format=torch.contiguous_format)
        out = torch.empty(B, T, H * D, dtype=q.dtype, device=q.device)
        L = N.lib()
        with _Device(q):
            work = torch.empty(L.ptb_paged_tree_work_floats(T, H, Hk, D), dtype=torch.float32, device=q.device)
            N.check(L.ptb_paged_attn_tree(q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(), B, T, H, Hk, D, lens.data_ptr(), N.ptr(nodes), N.ptr(mask), page_table.data_ptr(),
                                          page_table.stride(0), k_pages.shape[0], k_pages.data_ptr(), v_pages.data_ptr(), N.ptr(k_exp), N.ptr(v_exp), scale, work.data_ptr(),
                                          _status(q.device).data_ptr(), _on(q)), "paged_attention_tree")
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
    if not len(layers):
        return
    flat = []
    k0 = layers[0][0]
    Hk, D, quant = k0.shape[1], k0.shape[3], k0.dtype == E4M3
    for l in layers:
        k, v, ke, ve = l if len(l) == 4 else (*l, None, None)
        if k.shape != k0.shape or k.dtype != k0.dtype or v.shape != k0.shape or v.dtype != k0.dtype or not k.is_contiguous() or not v.is_contiguous() or k.device != k0.device \
                or v.device != k0.device or (ke is None) == quant or (ve is None) == quant:
            raise ValueError("paged_keep: layers need contiguous pools of one shape, type and device, with exponents if they are e4m3 and only then")
        if quant and not (ke.dtype == ve.dtype == torch.uint8 and ke.shape == ve.shape == k0.shape[:3] and ke.is_contiguous() and ve.is_contiguous()
                          and ke.device == ve.device == k0.device):
            raise ValueError("paged_keep: exponents are contiguous uint8 [page, kv head, 64]")
        flat += [k, v, ke, ve]
    _need(k0.dim() == 4 and k0.shape[2] == PAGE and path.dim() == 2, "paged_keep: pages [page, kv head, 64, D] and a path [B, T]")
    B, T = path.shape
    _index(path, k0, (B, T), "paged_keep: path")
    _index(lens, k0, (B,), "paged_keep: lens")
    _index(count, k0, (B,), "paged_keep: count")
    _need(page_table.dim() == 2 and page_table.shape[0] == B, f"paged_keep: a row of pages for each of {B} requests, not {list(page_table.shape)}")
    _index(page_table, k0, tuple(page_table.shape), "paged_keep: page_table")
    if k0.is_cuda:
        _need(D * k0.element_size() % 16 == 0, f"paged_keep: rows of 16-byte pieces are needed, not {D} x {k0.element_size()} bytes")
        ptrs = (C.c_void_p * len(flat))(*[t.data_ptr() if t is not None else None for t in flat])
        with _Device(k0):
            N.check(N.lib().ptb_paged_keep(ptrs, len(layers), B, T, Hk, D * k0.element_size(), k0.shape[0], lens.data_ptr(), path.data_ptr(), count.data_ptr(), page_table.data_ptr(),
                                           page_table.stride(0), _status(k0.device).data_ptr(), _on(k0)), "paged_keep")
        return
    for b in range(B):
        n = min(int(count[b]), T - 1)
        if n < 1:
            continue
        old, new = int(lens[b]) + path[b, 1:n + 1].long(), int(lens[b]) + torch.arange(1, n + 1)
        src, dst = _pages_of(page_table[b, old // PAGE], k0.shape[0]), _pages_of(page_table[b, new // PAGE], k0.shape[0])
        for t in flat:
            if t is not None:
                _as_bytes(t)[dst, :, new % PAGE] = _as_bytes(t)[src, :, old % PAGE]
