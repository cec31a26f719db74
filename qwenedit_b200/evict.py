"""Making a cached sequence smaller by what attention pays to its tokens.

``PagedKVPool`` evicts whole prefixes by time of use. A request whose own cache has grown too long keeps a part of it
instead: the tokens that got the most attention, beside the first ones and the latest (each layer and K/V head its
own). Three steps, each a call:

* ``attention_weights``  after an attention call: what every key got from that call's queries, added up over steps
* ``heaviest``           per layer and head, the positions to keep
* ``PagedKVPool.retain`` moves their K/V to other slots of the pool (``PagedKVPool.free`` gives the old ones back)

The kept tokens keep their keys' position encoding; a ``drafts.PagedBatch`` over the new slots attends to them.
No counterpart in the reference.
"""

from __future__ import annotations

import math

import torch

from qwenedit_b200 import _lib
from qwenedit_b200.drafts import DTYPES, DraftTree, PagedBatch, _check_apart, _check_pool, _check_rows, _view


def attention_weights(q: torch.Tensor, lse: torch.Tensor, cache: PagedBatch, tree: DraftTree, layer: int = 0,
                      k_draft: torch.Tensor | None = None, scale: float | None = None,
                      out: torch.Tensor | None = None, accumulate: bool = False) -> torch.Tensor:
    """The softmax weight every key got: out[b, g, j] = the sum, over request b's new tokens that see key j and the
    query heads of K/V head g, of exp(scale q . K_j - lse).

    The arguments of the attention call that made `lse` [Hq, T] fp32 (``drafts.tree_attention`` with the same cache
    and tree; or ``attention.paged_attention``, whose block of n queries is ``DraftTree([n])`` over a ``PagedBatch`` of
    one request, `full` where that call was not causal). Keys are the request's cached tokens, then, with `k_draft`,
    its new ones (in the tree's order). A token whose lse is +inf counts nothing (write it there to leave a rejected
    draft out), nor does one of -inf.

    Returns `out` [B, Hkv, W] fp32, by default as wide as the longest request needs: its slots, and with `k_draft` the
    tree's largest count. With `accumulate` the weights are added to what `out` holds (positions past a request's
    keys stay); else those positions get 0. The same inputs give the same bits. One launch on the current stream."""
    view = tree._view
    if view is None or view.cache is not cache:
        view = _view(cache, tree)
    key = (layer, scale, accumulate, q.shape, q.stride(), q.dtype, q.device,
           lse.shape, lse.stride(), lse.dtype, lse.device,
           None if k_draft is None else (k_draft.shape, k_draft.stride(), k_draft.dtype, k_draft.device),
           None if out is None else (out.shape, out.stride(), out.dtype, out.device))
    plan = view.plans.get(key)
    if plan is None:
        plan = view.keep(key, _WeightsPlan(view, tree, layer, q, lse, k_draft, scale, out, accumulate))
    device = plan.device
    if out is None:
        out = torch.empty(plan.shape, dtype=torch.float32, device=device)
    with _lib.on_device(device):
        args = plan.head + _WEIGHTS.pack(q.data_ptr(), *plan.q, cache.pool.kv.data_ptr() + plan.plane, plan.rows,
                                         0 if k_draft is None else k_draft.data_ptr(), *plan.draft, lse.data_ptr(),
                                         plan.lse, out.data_ptr(), *plan.tail)
        _lib.call("qe_attention_weights", args, _lib.stream_of(device))
    return out


_WEIGHTS = _lib.ATTENTION_WEIGHTS


class _WeightsPlan:
    """The checked layouts of an ``attention_weights`` call as the numbers its C arguments need."""

    def __init__(self, view, tree, layer, q, lse, k_draft, scale, out, accumulate):
        cache = view.cache
        pool = _check_pool(cache, layer)
        kv, device, heads_kv, d = pool.kv, pool.device, pool.heads, pool.head_dim
        if q.dim() != 3 or q.shape[1] % heads_kv or q.shape[1] == 0:
            raise ValueError(f"q must be [tokens, heads, {d}], its heads a multiple of the pool's {heads_kv}")
        total, heads_q, width = tree.total, q.shape[1], cache.max_length
        _check_rows("q", q, total, heads_q, d, kv.dtype, device)
        self.draft = (0, 0)
        if k_draft is not None:
            _check_rows("k_draft", k_draft, total, heads_kv, d, kv.dtype, device)
            self.draft = (2 * k_draft.stride(0), 2 * k_draft.stride(1))
            width += tree.max_nodes
        if lse.device != device or lse.dtype != torch.float32 or lse.dim() != 2 or lse.shape[0] != heads_q or \
                lse.shape[1] < total or (lse.shape[1] > 1 and lse.stride(1) != 1):
            raise ValueError(f"lse must be [{heads_q}, at least {total}] float32 on {device} with contiguous rows")
        if out is None:
            if accumulate:
                raise ValueError("accumulate needs `out`")
            strides = (heads_kv * width, width)
        else:
            strides = out.stride()
            if out.device != device or out.dtype != torch.float32 or out.dim() != 3 or out.shape[0] != cache.batch or \
                    out.shape[1] != heads_kv or out.shape[2] < width or (out.shape[2] > 1 and strides[2] != 1):
                raise ValueError(f"out must be [{cache.batch}, {heads_kv}, at least {width}] float32 on {device} with "
                                 "contiguous rows")
            width = out.shape[2]
            _check_apart(out)
        self.device, self.head, self.shape, self.lse = device, view.batch, (cache.batch, heads_kv, width), lse.stride(0)
        self.q, self.plane, self.rows = (2 * q.stride(0), 2 * q.stride(1)), 2 * layer * kv.stride(0), pool.rows
        self.tail = (strides[0], strides[1], width, pool._err.data_ptr(), heads_q, heads_kv, d, DTYPES[kv.dtype],
                     1 if accumulate else 0, 1.0 / math.sqrt(d) if scale is None else float(scale))


def heaviest(weights: torch.Tensor, budget: int, lengths: torch.Tensor | None = None, sinks: int = 0,
             recent: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """The positions a cache of `budget` tokens keeps, per row of `weights` [..., N] (fp32; up to three leading
    dimensions, e.g. layers and K/V heads): the first `sinks`, the last `recent` and, of the others, the heaviest; of
    equal weights the lowest position first, NaN as -inf.

    `lengths` (int32 on the device, broadcast to the leading dimensions): how many positions a row holds; default N.
    Returns (keep [..., budget] int32 in rising order, the kept positions' weights [..., budget] fp32); where a row
    holds fewer than `budget` positions it keeps them all and the rest is -1 and 0. One launch."""
    budget, sinks, recent = int(budget), int(sinks), int(recent)
    if weights.device.type != "cuda":
        raise RuntimeError("heaviest runs only on CUDA devices (no CPU path)")
    if weights.dtype != torch.float32 or not 1 <= weights.dim() <= 4:
        raise ValueError("weights must be float32 with one to four dimensions")
    if budget < 0 or sinks < 0 or recent < 0 or sinks + recent > budget:
        raise ValueError(f"budget {budget} must hold the {sinks} first and {recent} last positions")
    lead = weights.shape[:-1]
    if weights.shape[-1] > 1 and weights.stride(-1) != 1:
        weights = weights.contiguous()
    if lengths is not None:
        if lengths.device != weights.device or lengths.dtype != torch.int32:
            raise ValueError(f"lengths must be int32 on {weights.device}")
        if lengths.shape != lead or not lengths.is_contiguous():
            lengths = lengths.broadcast_to(lead).contiguous()
    n = [1] * (3 - len(lead)) + list(lead)
    s = [0] * (3 - len(lead)) + list(weights.stride()[:-1])
    keep = torch.empty((*lead, budget), dtype=torch.int32, device=weights.device)
    kept = torch.empty_like(keep, dtype=torch.float32)
    with _lib.on_device(weights.device):
        _lib.call("qe_heaviest", weights.data_ptr(), *n, *s, weights.shape[-1],
                  None if lengths is None else lengths.data_ptr(), budget, sinks, recent, keep.data_ptr(),
                  kept.data_ptr(), _lib.stream_of(weights.device))
    return keep, kept
