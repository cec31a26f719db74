"""Decoding over the pooled caches: attention of a batch's newest tokens, one or a tree of drafted ones a request.

``attention.paged_attention`` attends with one request's block of queries (an edit's latent tokens, a prompt's tail).
A program that writes text on the encoder's pool works on many requests at once, each with its own cached length and
a few new tokens: the last one written, a chain of guesses, or a tree of them whose nodes see their ancestors only.

* ``PagedBatch``   the cached tokens of the requests: slots of a ``PagedKVPool`` as device block tables, and lengths
* ``DraftTree``    the new tokens of the requests: counts, and what each sees of the others
* ``tree_attention`` their attention, one layer (``qe_tree_attention``)

Lengths, tables and masks live in device memory and are read when the kernels run, so a captured CUDA graph replays
with what they hold then (``PagedBatch.set_lengths``, ``DraftTree.set_parents``). No counterpart in the reference.
"""

from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

from qwenedit_b200 import _lib

DTYPES = {torch.bfloat16: 1, torch.float16: 2}
HEAD_DIMS = (64, 128)


def _to_device(host: np.ndarray, device: torch.device) -> torch.Tensor:
    t = torch.from_numpy(host)
    if device.type != "cuda":
        return t.to(device)
    if torch.cuda.is_current_stream_capturing():
        # the copy would be replayed from host memory that is no longer these values
        raise RuntimeError("values from the host cannot go into a captured graph: set them outside of it")
    return t.pin_memory().to(device, non_blocking=True)


class PagedBatch:
    """Cached tokens of a batch of requests: `indices`, one slot tensor of `pool` per request (what ``match``,
    ``alloc`` or ``cat_slots`` returned; None or empty: no room), and how many of them hold tokens now (`lengths`,
    default all). With a page size above 1 the slots must be whole-page runs. Slots past a request's length are room
    to grow: ``set_lengths`` after writing there. The same slots may stand in several requests (a shared prefix)."""

    def __init__(self, pool, indices, lengths=None):
        self.pool = pool
        self.indices = list(indices)
        self.batch = len(self.indices)
        P = pool.page_size
        tables = []
        for i, ix in enumerate(self.indices):
            host = np.empty(0, np.int64) if ix is None else pool._host_slots(ix)
            if len(host) and (host.min() < 0 or host.max() >= pool.rows):
                raise ValueError(f"slots of request {i} outside the pool's {pool.rows} rows")
            pages = host[::P] // P
            at = np.arange(len(host), dtype=np.int64)
            if not np.array_equal(host, pages[at // P] * P + at % P):
                raise ValueError(f"slots of request {i} are not whole-page runs (page_size {P})")
            tables.append((pages, len(host)))
        self.room = [n for _, n in tables]
        self.max_length, self.sum_length = max(self.room, default=0), sum(self.room)
        self.table_width = max((len(pages) for pages, _ in tables), default=0)
        table = np.full((self.batch, self.table_width), -1, np.int32)
        for i, (pages, _) in enumerate(tables):
            table[i, : len(pages)] = pages
        self._tables = _to_device(table, pool.device)
        pool.h2d_bytes += table.nbytes
        self._lengths = torch.zeros(self.batch, dtype=torch.int32, device=pool.device)
        self.set_lengths(self.room if lengths is None else lengths)

    @property
    def tables(self) -> torch.Tensor:
        """[batch, table_width] int32 page ids on the device (in place only: the kernels keep reading this memory)."""
        return self._tables

    @property
    def lengths(self) -> torch.Tensor:
        """[batch] int32 cached tokens on the device (in place only; what a device-side loop may add to)."""
        return self._lengths

    def set_lengths(self, lengths) -> None:
        """The cached tokens of each request from now on (on the current stream), at most its slots."""
        host = [int(n) for n in lengths]
        if len(host) != self.batch or any(not 0 <= n <= room for n, room in zip(host, self.room)):
            raise ValueError(f"lengths must be {self.batch} counts within the requests' slots {self.room}")
        self.lengths.copy_(_to_device(np.asarray(host, np.int32), self.pool.device), non_blocking=True)


class DraftTree:
    """New tokens ("nodes") of a batch of requests: `counts[b]` of them for request b, laid out one request after the
    other. What a node sees of its request's nodes:

    * `parents` None: a chain, node i sees nodes 0 .. i (one token a request: ``DraftTree([1] * batch)``); with
      `full`, every node of the request;
    * `parents` (a sequence, or an int32 tensor on the device, over all nodes): itself and its ancestors; the parent's
      index within the request, -1 for a node that follows the cache. Parents come before their children;
    * `visible`: one [n, n] bool array per request, row i = what node i sees (it may be nothing).
    """

    CHAIN, MASKS, FULL = 0, 1, 2

    def __init__(self, counts, parents=None, visible=None, full: bool = False, device="cuda"):
        self.counts = [int(n) for n in counts]
        if any(n < 0 for n in self.counts):
            raise ValueError("counts must not be negative")
        if (parents is not None) + (visible is not None) + bool(full) > 1:
            raise ValueError("parents, visible and full exclude each other")
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.batch = len(self.counts)
        starts = np.zeros(self.batch + 1, np.int64)
        np.cumsum(self.counts, out=starts[1:])
        if starts[-1] >= 1 << 31:
            raise ValueError("too many nodes")
        self._host_starts = starts
        self.total, self.max_nodes = int(starts[-1]), max(self.counts, default=0)
        self._starts = _to_device(starts.astype(np.int32), self.device)
        self.mode, self._masks, self.words = (self.FULL if full else self.CHAIN), None, 0
        self._err = None
        self._view = None
        if parents is not None or visible is not None:
            self.mode, self.words = self.MASKS, max(1, -(-self.max_nodes // 32))
            self._masks = torch.zeros(self.total, self.words, dtype=torch.int32, device=self.device)
        if parents is not None:
            self.set_parents(parents)
        if visible is not None:
            self._set_visible(visible)

    @property
    def starts(self) -> torch.Tensor:
        """[batch + 1] int32: the first node of each request, on the device (for kernels to read: the counts are fixed, and
        a call's outputs have their rows)."""
        return self._starts

    @property
    def masks(self) -> torch.Tensor | None:
        """[total, words] int32 bit masks on the device (in place only); None for a chain or `full`."""
        return self._masks

    def set_parents(self, parents) -> None:
        """Another tree of the same counts: rebuilds the masks in place, one launch on the current stream (with a
        device tensor nothing is copied from the host). A device tensor's parents are checked on the device: one
        outside [-1, node) counts as -1 and shows in ``device_errors``."""
        if self.mode != self.MASKS:
            raise ValueError("this DraftTree was made without parents")
        if isinstance(parents, torch.Tensor) and parents.device.type == "cuda":
            if parents.device != self.device or parents.dtype != torch.int32 or parents.numel() != self.total:
                raise ValueError(f"parents must be {self.total} int32 values on {self.device}")
            dev = parents.contiguous()
        else:
            host = np.asarray(parents.numpy() if isinstance(parents, torch.Tensor) else parents, np.int64).reshape(-1)
            at = np.arange(self.total) - np.repeat(self._host_starts[:-1], self.counts)
            if len(host) != self.total or bool((host < -1).any()) or bool((host >= at).any()):
                raise ValueError(f"parents must be {self.total} indices within the requests, each before its child "
                                 "(-1: follows the cache)")
            dev = _to_device(host.astype(np.int32), self.device)
        if self.device.type != "cuda":
            raise RuntimeError("a DraftTree's masks are built on CUDA devices (no CPU path)")
        if self._err is None:
            self._err = torch.zeros(1, dtype=torch.int32, device=self.device)
        with _lib.on_device(self.device):
            _lib.call("qe_tree_masks", dev.data_ptr(), self.starts.data_ptr(), self.batch, self.total, self.max_nodes,
                      self.words, self.masks.data_ptr(), self._err.data_ptr(), _lib.stream_of(self.device))

    def _set_visible(self, visible) -> None:
        visible = list(visible)
        words = np.zeros((self.total, self.words), np.uint32)
        if len(visible) != self.batch:
            raise ValueError(f"visible must hold one array for each of the {self.batch} requests")
        for b, v in enumerate(visible):
            v = v.cpu().numpy() if isinstance(v, torch.Tensor) else np.asarray(v)
            n = self.counts[b]
            if v.shape != (n, n) or v.dtype != np.bool_:
                raise ValueError(f"visible[{b}] must be a bool array of [{n}, {n}]")
            bits = np.zeros((n, self.words * 32), np.uint32)
            bits[:, :n] = v
            lo = int(self._host_starts[b])
            words[lo : lo + n] = (bits.reshape(n, self.words, 32) << np.arange(32, dtype=np.uint32)).sum(
                -1, dtype=np.uint32)
        self.masks.copy_(_to_device(words.view(np.int32), self.device), non_blocking=True)

    def device_errors(self) -> int:
        """Non-zero when ``set_parents`` met a bad parent on the device since the last call (reads the flag)."""
        if self._err is None:
            return 0
        value = int(self._err.item())
        self._err.zero_()
        return value


class _View:
    """The C view of a cache and a tree (``qe_draft_batch`` as bytes), and what the calls made with them have checked
    and worked out, by the layouts of their tensors."""

    __slots__ = ("cache", "batch", "plans")

    def __init__(self, cache, batch):
        self.cache, self.batch, self.plans = cache, batch, {}

    def keep(self, key, plan):
        if len(self.plans) >= 1024:  # a program whose layouts never repeat
            self.plans.clear()
        self.plans[key] = plan
        return plan


def _view(cache: PagedBatch, tree: DraftTree) -> _View:
    """Kept with the tree while the two stay together."""
    kept = tree._view
    if kept is not None and kept.cache is cache:
        return kept
    if cache.batch != tree.batch:
        raise ValueError(f"the cache holds {cache.batch} requests, the tree {tree.batch}")
    if cache.pool.device != tree.device:
        raise ValueError(f"the cache is on {cache.pool.device}, the tree on {tree.device}")
    batch = _lib.DRAFT_BATCH.pack(tree.starts.data_ptr(), cache.lengths.data_ptr(), cache.tables.data_ptr(),
                                  0 if tree.masks is None else tree.masks.data_ptr(), cache.batch, cache.table_width,
                                  cache.pool.page_size, tree.words, tree.mode, tree.total, tree.max_nodes,
                                  cache.max_length, cache.sum_length)
    view = tree._view = _View(cache, batch)
    return view  # (the tree's may be another thread's by now)


def _check_rows(name: str, t: torch.Tensor, n: int, heads: int, head_dim: int, dtype, device) -> None:
    if t.device != device or device.type != "cuda":
        raise ValueError(f"{name} must be a CUDA tensor on {device}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, as the pool")
    if t.dim() != 3 or t.shape[0] < n or t.shape[1] != heads or t.shape[2] != head_dim or t.stride(2) != 1:
        raise ValueError(f"{name} must be [at least {n} tokens, {heads} heads, {head_dim}] with contiguous head rows")


def _check_apart(t: torch.Tensor) -> None:
    """An output's rows (its last dimension) must not share memory: several of them are written at once."""
    end = t.shape[-1]
    for step, n in sorted((t.stride(i), t.shape[i]) for i in range(t.dim() - 1) if t.shape[i] > 1):
        if step < end:
            raise ValueError("out must not have rows that overlap")
        end += step * (n - 1)


def _check_pool(cache: PagedBatch, layer: int):
    pool = cache.pool
    if pool.kv.dtype not in DTYPES or pool.head_dim not in HEAD_DIMS:
        raise ValueError(f"the pool must hold bf16 or fp16 heads of {' or '.join(map(str, HEAD_DIMS))}")
    if not 0 <= layer < pool.layers:
        raise ValueError(f"layer {layer} outside the pool's {pool.layers}")
    return pool


def tree_attention(q: torch.Tensor, cache: PagedBatch, tree: DraftTree, layer: int = 0,
                   k_draft: torch.Tensor | None = None, v_draft: torch.Tensor | None = None,
                   scale: float | None = None, out: torch.Tensor | None = None, return_lse: bool = False):
    """softmax(q K^T * scale) V of every new token over [its request's cached tokens; the new tokens it sees].

    q [T, Hq, D] in the pool's type (bf16 or fp16, D 64 or 128), T >= ``tree.total`` rows in the tree's order; Hq a
    multiple of the pool's Hkv (query head h reads K/V head h // (Hq // Hkv)); k_draft / v_draft [T, Hkv, D], the new
    tokens' own K/V (both None: the new tokens see the cache only, e.g. when their K/V were written to the pool and
    counted in the lengths). Any strides that are multiples of 16 bytes with contiguous head rows. Returns out
    [T, Hq, D], and with `return_lse` the log-sum-exp [Hq, tree.total] fp32 of the scaled scores, which
    ``evict.attention_weights`` takes. A token that sees nothing gets zeros and -inf; rows of `out` past the tree's
    are left as they were (zeros where the call makes `out`). Runs on the current stream, without synchronising."""
    view = tree._view
    if view is None or view.cache is not cache:
        view = _view(cache, tree)
    key = (layer, scale, q.shape, q.stride(), q.dtype, q.device,
           None if k_draft is None else (k_draft.shape, k_draft.stride(), k_draft.dtype, k_draft.device),
           None if v_draft is None else (v_draft.shape, v_draft.stride(), v_draft.dtype, v_draft.device),
           None if out is None else (out.shape, out.stride(), out.dtype, out.device))
    plan = view.plans.get(key)
    if plan is None:
        plan = view.keep(key, _TreePlan(view, tree, layer, q, k_draft, v_draft, scale, out))
    if out is None:
        out = (torch.empty_like if plan.exact else torch.zeros_like)(q, memory_format=torch.contiguous_format)
    device, plane = plan.device, cache.pool.kv.data_ptr() + plan.plane
    lse = torch.empty_strided(plan.lse, plan.lse_strides, dtype=torch.float32, device=device) if return_lse else None
    with _lib.on_device(device):
        work = torch.empty(plan.work, dtype=torch.uint8, device=device) if plan.work else None
        args = plan.head + _TREE.pack(
            q.data_ptr(), *plan.q, plane, plane + plan.to_v, plan.rows, 0 if k_draft is None else k_draft.data_ptr(),
            0 if v_draft is None else v_draft.data_ptr(), *plan.draft, out.data_ptr(), *plan.out,
            0 if lse is None else lse.data_ptr(), 0 if work is None else work.data_ptr(), *plan.tail)
        _lib.call("qe_tree_attention", args, _lib.stream_of(device))
    return (out, lse) if return_lse else out


_TREE = _lib.TREE_ATTENTION


class _TreePlan:
    """The checked layouts of a ``tree_attention`` call as the numbers its C arguments need."""

    def __init__(self, view, tree, layer, q, k_draft, v_draft, scale, out):
        pool = _check_pool(view.cache, layer)
        kv, device, heads_kv, d = pool.kv, pool.device, pool.heads, pool.head_dim
        if q.dim() != 3 or q.shape[1] % heads_kv or q.shape[1] == 0:
            raise ValueError(f"q must be [tokens, heads, {d}], its heads a multiple of the pool's {heads_kv}")
        if (k_draft is None) != (v_draft is None):
            raise ValueError("k_draft and v_draft go together")
        total, heads_q = tree.total, q.shape[1]
        _check_rows("q", q, total, heads_q, d, kv.dtype, device)
        self.draft = (0, 0)
        if k_draft is not None:
            _check_rows("k_draft", k_draft, total, heads_kv, d, kv.dtype, device)
            _check_rows("v_draft", v_draft, total, heads_kv, d, kv.dtype, device)
            if k_draft.stride() != v_draft.stride():
                raise ValueError("k_draft and v_draft must have the same strides")
            self.draft = (2 * k_draft.stride(0), 2 * k_draft.stride(1))
        if out is not None:
            _check_rows("out", out, total, heads_q, d, kv.dtype, device)
            _check_apart(out)
        self.device, self.exact, self.head = device, q.shape[0] == total, view.batch
        self.q, self.rows = (2 * q.stride(0), 2 * q.stride(1)), pool.rows
        self.plane, self.to_v = 2 * layer * kv.stride(0), 2 * kv.stride(1)
        self.out = (2 * heads_q * d, 2 * d) if out is None else (2 * out.stride(0), 2 * out.stride(1))
        self.lse, self.lse_strides = (heads_q, total), (total, 1)
        heads = (heads_q, heads_kv, d, DTYPES[kv.dtype])
        size = ctypes.c_int64()
        with _lib.on_device(device):
            _lib.call("qe_tree_attention_workspace", view.batch + _TREE.pack(*[0] * 17, *heads, 1.0),
                      ctypes.byref(size))
        self.work = size.value
        self.tail = (size.value, pool._err.data_ptr(), *heads, 1.0 / math.sqrt(d) if scale is None else float(scale))
