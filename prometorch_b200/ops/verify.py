"""Which drafted tokens a target model keeps: :func:`verify_drafts`, the decision between two steps of speculative decoding, on the device and from given random numbers.

With tokens proposed outright (an n-gram look-up, the best few of a draft model) several may hang on one parent: they are tried in order, each accepted with its
probability under what the rejected ones before it have left of the target's distribution.  With a draft model's probabilities the drafts are a chain, accepted with probability
min(1, p / q), and a rejection draws from max(p - q, 0).  Either way the tokens that come out are distributed as the target's own.

CUDA tensors go through csrc/verify.cu (logits read once, the draw's row in fp64); CPU tensors take the plain form below."""
from __future__ import annotations

import ctypes as C
import functools
from typing import Optional, Tuple

import torch

from .. import _native as N
from .paged_tree import _index, _launch

MAX_NODES = 64
MAX_VOCAB = 442368          # on the GPU: what a cluster's shared memory holds
MAX_TEMPERATURE = 2.0 ** 126


@N.register_decls
def _decls(L):
    vp, ci, ll = C.c_void_p, C.c_int, C.c_longlong
    if hasattr(L, "ptb_verify_drafts"):
        L.ptb_verify_drafts.argtypes = [vp, ci, ll, ll, vp, ll, ll, vp, vp, vp, vp, vp, vp, vp, vp, vp, ci, ci, ci, vp]
        L.ptb_verify_drafts.restype = ci
        L.ptb_verify_work_bytes.argtypes = [ci, ci, ci]
        L.ptb_verify_work_bytes.restype = ll


def _floats(t: torch.Tensor, dev: torch.device, at: int, shape: tuple, name: str) -> None:
    if t.dtype is not torch.float32 or t.shape != shape or not t.is_contiguous() or t.get_device() != at:
        raise ValueError(f"verify_drafts: {name} is a contiguous fp32 tensor {list(shape)} on {dev}, not {t.dtype} {list(t.shape)} on {t.device}")


@functools.lru_cache(maxsize=1024)
def _work_bytes(B: int, T: int, V: int) -> int:
    return N.lib().ptb_verify_work_bytes(B, T, V)


def verify_drafts(logits: torch.Tensor, tokens: torch.Tensor, u: torch.Tensor, temperature: torch.Tensor, parents: Optional[torch.Tensor] = None,
                  nodes: Optional[torch.Tensor] = None, draft_probs: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``logits [B, T, V]`` (fp32 or bf16): what the target says behind each of a request's T nodes; node 0 is the latest token, the others are drafted.  ``tokens [B, T]`` (int32):
    their ids; ``parents [B, T]`` (int32): a node before the node, -1 for the first (None: a chain); ``nodes [B]`` (int32): how many are there (None: all).  ``u [B, T]`` (fp32 in
    [0, 1)): node i's number decides on it, the first one's draws the last token.  ``temperature [B]`` (fp32): 0 or below takes the arg-max, of equals the lowest id; above 2^126
    (infinity too) counts as 2^126, a uniform row for logits of any ordinary size.
    ``draft_probs [B, T, V]`` (fp32, chains only): row i is what the node behind node i was drawn from.

    Returns ``(path, count, out)``, int32: ``path [B, T]`` the accepted nodes, the first one among them, -1 behind; ``count [B]`` how many drafted tokens were accepted (-1 for a
    request without nodes); ``out [B, T]`` their tokens and then the one that the target adds, -1 behind.

    On the GPU a batch has up to 65536 nodes and a row up to 442368 tokens.

    A logit of -inf (or NaN) is a token of probability zero; where nothing is left to draw from, the arg-max of the row is taken.  Siblings with one token count
    once.  A token outside the vocabulary is rejected, a node whose parent does not come before it is never reached."""
    if logits.dim() != 3 or logits.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"verify_drafts: fp32 or bf16 logits [B, T, V] are needed, not {logits.dtype} {list(logits.shape)}")
    B, T, V = logits.shape
    dev, home = logits.device, logits.get_device()
    if not 1 <= T <= MAX_NODES or V < 1:
        raise ValueError(f"verify_drafts: 1 to {MAX_NODES} nodes a request and a vocabulary, not {T} and {V}")
    _index(tokens, dev, home, (B, T), "verify_drafts: tokens")
    if parents is not None:
        _index(parents, dev, home, (B, T), "verify_drafts: parents")
        if draft_probs is not None:
            raise ValueError("verify_drafts: draft probabilities go with chains")
    if nodes is not None:
        _index(nodes, dev, home, (B,), "verify_drafts: nodes")
    _floats(u, dev, home, (B, T), "u")
    _floats(temperature, dev, home, (B,), "temperature")
    if draft_probs is not None and (draft_probs.dtype != torch.float32 or draft_probs.shape != logits.shape or draft_probs.get_device() != home):
        raise ValueError(f"verify_drafts: draft_probs are fp32 {[B, T, V]} on {dev}, not {draft_probs.dtype} {list(draft_probs.shape)} on {draft_probs.device}")
    if logits.is_cuda:
        if logits.stride(2) != 1:
            logits = logits.contiguous()
        p_batch = p_row = 0
        if draft_probs is not None:
            if draft_probs.stride(2) != 1:
                draft_probs = draft_probs.contiguous()
            p_batch, p_row, _ = draft_probs.stride()
        l_batch, l_row, _ = logits.stride()
        path, out = torch.empty(2, B, T, dtype=torch.int32, device=dev).unbind(0)
        count = torch.empty(B, dtype=torch.int32, device=dev)
        L = N.lib()
        work = torch.empty(_work_bytes(B, T, V), dtype=torch.uint8, device=dev)
        rc = _launch(home, L.ptb_verify_drafts, logits.data_ptr(), int(logits.dtype is torch.bfloat16), l_batch, l_row, N.ptr(draft_probs), p_batch, p_row, tokens.data_ptr(),
                     N.ptr(parents), N.ptr(nodes), u.data_ptr(), temperature.data_ptr(), work.data_ptr(), path.data_ptr(), count.data_ptr(), out.data_ptr(), B, T, V)
        if rc:
            N.check(rc, "verify_drafts")
        return path, count, out
    return verify_drafts_reference(logits, tokens, u, temperature, parents, nodes, draft_probs)


def verify_drafts_reference(logits, tokens, u, temperature, parents=None, nodes=None, draft_probs=None):
    """The walk, request by request in fp64: the CPU path."""
    B, T, V = logits.shape
    path, out = torch.full((B, T), -1, dtype=torch.int32), torch.full((B, T), -1, dtype=torch.int32)
    count = torch.full((B,), -1, dtype=torch.int32)
    for b in range(B):
        n = T if nodes is None else max(0, min(int(nodes[b]), T))
        if n == 0:
            continue
        temp = min(float(temperature[b]), MAX_TEMPERATURE)
        up = [-1] + [(i - 1 if parents is None else int(parents[b, i])) for i in range(1, n)]
        tok = tokens[b].tolist()

        def weights(i):
            x = logits[b, i].double()
            x = torch.where(torch.isnan(x), torch.full_like(x, -float("inf")), x)
            best = x.max()
            first = int((x == best).nonzero()[0])
            w = torch.where(x == best, torch.ones_like(x), torch.exp((x - best) / (temp if temp > 0 else 1.0)))
            return torch.where(x == -float("inf"), torch.zeros_like(x), w), first
        at, walk = 0, [0]
        while True:
            w, first = weights(at)
            left = w.clone()
            kids = [c for c in range(at + 1, n) if up[c] == at]
            nxt = None
            for c in kids:
                x = tok[c]
                mine = float(left[x]) if 0 <= x < V else 0.0
                if temp > 0:
                    q = 1.0 if draft_probs is None else float(draft_probs[b, at, x]) if 0 <= x < V else 0.0
                    take = float(u[b, c]) * float(left.sum()) * q < mine
                else:
                    take = x == first
                if take:
                    nxt = c
                    break
                if draft_probs is None and 0 <= x < V:
                    left[x] = 0
            if nxt is None:
                break
            at = nxt
            walk.append(at)
        if temp > 0:
            if draft_probs is not None and kids:
                left = (w / w.sum() - draft_probs[b, at].double()).clamp_min(0)
            c = left.cumsum(0)
            if float(c[-1]) > 0:
                over = (c > float(u[b, 0]) * float(c[-1])).nonzero()
                last = int(over[0]) if len(over) else int((left > 0).nonzero()[-1])
            else:
                last = first
        else:
            last = first
        k = len(walk)
        path[b, :k] = torch.tensor(walk, dtype=torch.int32)
        count[b] = k - 1
        out[b, :k] = torch.tensor([tok[i] for i in walk[1:]] + [last], dtype=torch.int32)
    return path, count, out
