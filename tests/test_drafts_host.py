"""What the decoding and cache-eviction operators refuse, on the CPU: bad shapes, types, counts and slots raise before
any launch, and the C entry points reject bad arguments without touching the GPU."""

import ctypes

import numpy as np
import pytest
import torch

from qwenedit_b200 import _lib
from qwenedit_b200.drafts import DraftTree, PagedBatch, _check_apart, _view, tree_attention
from qwenedit_b200.evict import attention_weights, heaviest
from qwenedit_b200.paged import PagedKVPool, cat_slots


def _pool(page=4, dtype=torch.bfloat16, d=64, heads=2):
    return PagedKVPool("host", 1, heads, d, 32 * 2 * heads * d * 2, dtype, "cpu", page_size=page)


def test_batch_needs_whole_pages_in_the_pool():
    pool = _pool()
    run = torch.arange(8, 14)
    b = PagedBatch(pool, [run, None, torch.empty(0, dtype=torch.int64)])
    assert b.tables.tolist() == [[2, 3], [-1, -1], [-1, -1]] and b.lengths.tolist() == [6, 0, 0]
    assert (b.max_length, b.sum_length, b.table_width) == (6, 6, 2)
    for bad in (torch.tensor([8, 9, 11]), torch.tensor([9, 10]), torch.tensor([8, 9, 10, 11, 13])):
        with pytest.raises(ValueError, match="whole-page runs"):
            PagedBatch(pool, [bad])
    for bad in (torch.tensor([-4, -3]), torch.arange(pool.rows - 1, pool.rows + 1)):
        with pytest.raises(ValueError, match="outside the pool"):
            PagedBatch(pool, [bad])
    for lengths in ([7, 0, 0], [-1, 0, 0], [1, 1, 0], [1, 0]):
        with pytest.raises(ValueError, match="lengths"):
            PagedBatch(pool, [run, None, None], lengths)
    assert PagedBatch(_pool(page=1), [torch.tensor([5, 3, 9])]).tables.tolist() == [[5, 3, 9]]


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_slots_written_in_place_are_read_again(dtype):
    pool = _pool(page=1)
    slots = torch.tensor([5, 3, 9], dtype=dtype)
    assert PagedBatch(pool, [slots]).tables.tolist() == [[5, 3, 9]]
    slots[1] = 7
    assert PagedBatch(pool, [slots]).tables.tolist() == [[5, 7, 9]]
    with torch.inference_mode():
        slots.add_(1)
        assert PagedBatch(pool, [slots]).tables.tolist() == [[6, 8, 10]]
    tail = slots[1:]
    assert PagedBatch(pool, [tail]).tables.tolist() == [[8, 10]]
    slots[2] = 1  # through the tensor that it is a view of
    assert PagedBatch(pool, [tail]).tables.tolist() == [[8, 1]]
    slots[0] = pool.rows
    with pytest.raises(ValueError, match="outside the pool"):
        PagedBatch(pool, [slots])
    with torch.inference_mode():  # tensors that do not count their changes
        own = torch.tensor([5, 3], dtype=dtype)
        assert PagedBatch(pool, [own]).tables.tolist() == [[5, 3]]
        own[0] = 4
        assert PagedBatch(pool, [own]).tables.tolist() == [[4, 3]]


@pytest.mark.parametrize("inference", [False, True])
def test_allocated_slots_written_in_place_are_read_again(inference):
    pool = _pool(page=4)
    with torch.inference_mode(inference):
        a = pool.alloc(8)
        both = cat_slots(a, pool.alloc(4))
        assert PagedBatch(pool, [both]).tables.tolist() == [[1, 2, 3]]
        a.copy_(a.flip(0).reshape(2, 4).flip(1).reshape(-1))  # its pages the other way round
        both[:8] = a
        assert PagedBatch(pool, [a, both, cat_slots(both, a)]).tables.tolist() == [
            [2, 1, -1, -1, -1], [2, 1, 3, -1, -1], [2, 1, 3, 2, 1]]
        pool.insert(np.arange(12), both, 0)
        hit = pool.match(np.arange(12))
        assert hit.indices.tolist() == both.tolist()
        hit.indices[:4] = 0
        assert pool.match(np.arange(12)).indices.tolist() == both.tolist()


def test_tree_counts_parents_and_masks():
    t = DraftTree([2, 0, 3], device="cpu")
    assert t.starts.tolist() == [0, 2, 2, 5] and (t.total, t.max_nodes, t.batch) == (5, 3, 3)
    with pytest.raises(ValueError, match="negative"):
        DraftTree([1, -1], device="cpu")
    with pytest.raises(ValueError, match="exclude"):
        DraftTree([2], [-1, 0], full=True, device="cpu")
    with pytest.raises(ValueError, match="made without parents"):
        t.set_parents([-1] * 5)
    for parents in ([-1], [-1, 1], [0, 0], [-2, 0], [-1, 0, 1]):
        with pytest.raises(ValueError, match="before its child"):
            DraftTree([2], parents, device="cpu")
    with pytest.raises(ValueError, match="before its child"):
        DraftTree([1, 2], [-1, -1, 1], device="cpu")  # indices count within the request
    with pytest.raises(RuntimeError, match="CUDA"):
        DraftTree([2], [-1, 0], device="cpu")
    see = np.zeros((40, 40), bool)
    see[3, [0, 31, 32, 39]] = True
    m = DraftTree([1, 40], visible=[np.ones((1, 1), bool), see], device="cpu").masks
    assert m.shape == (41, 2) and m[0].tolist() == [1, 0] and m[1].tolist() == [0, 0]
    assert m[4].tolist() == [1 - 2**31, 1 | 1 << 7]
    for bad in ([see], [np.ones((1, 1), bool), see[:3]], [np.ones((1, 1), np.int8), see]):
        with pytest.raises(ValueError, match="visible"):
            DraftTree([1, 40], visible=bad, device="cpu")


def _args(pool=None, n=3, hq=4, dtype=torch.bfloat16):
    pool = _pool() if pool is None else pool
    rand = lambda h: torch.zeros(n, h, pool.head_dim, dtype=dtype)  # noqa: E731
    return rand(hq), PagedBatch(pool, [torch.arange(4, 8)]), DraftTree([n], device="cpu"), 0, rand(pool.heads), rand(pool.heads)


def test_a_tree_shared_by_threads_with_their_own_caches():
    """Between one thread's storing of its view with the tree and its next line another thread stores its own."""
    pool = _pool()
    ours, theirs = PagedBatch(pool, [torch.arange(4, 8)]), PagedBatch(pool, [torch.arange(8, 20)])

    class Shared(DraftTree):
        @property
        def _view(self):
            return self.stored

        @_view.setter
        def _view(self, view):
            self.stored = view if view is None else _view(theirs, DraftTree([3], device="cpu"))

    tree = Shared([3], device="cpu")
    view = _view(ours, tree)
    assert view.cache is ours and view.batch == _view(ours, tree).batch
    assert tree.stored.cache is theirs


def test_tree_attention_refuses_before_any_launch():
    with pytest.raises(ValueError, match="CUDA tensor"):
        tree_attention(*_args())
    with pytest.raises(ValueError, match="multiple of the pool's 2"):
        tree_attention(*_args(hq=3))
    q, cache, tree, layer, kn, vn = _args()
    with pytest.raises(ValueError, match="layer 1 outside"):
        tree_attention(q, cache, tree, 1, kn, vn)
    with pytest.raises(ValueError, match="bf16 or fp16"):
        tree_attention(*_args(_pool(dtype=torch.float32)))
    with pytest.raises(ValueError, match="bf16 or fp16 heads"):
        tree_attention(*_args(_pool(d=32)))


def test_outputs_must_not_overlap_themselves():
    x = torch.zeros(10_000)
    for sizes, strides in [((3, 2, 64), (128, 64, 1)), ((3, 2, 64), (64, 192, 1)), ((2, 3, 50), (300, 64, 1)),
                           ((1, 1, 64), (0, 0, 1)), ((1, 4, 64), (3, 64, 1)), ((0, 4, 64), (0, 64, 1))]:
        _check_apart(x.as_strided(sizes, strides))
    for sizes, strides in [((3, 2, 64), (64, 64, 1)), ((3, 2, 64), (0, 64, 1)), ((3, 2, 64), (128, 63, 1)),
                           ((3, 2, 64), (64, 128, 1)), ((2, 3, 50), (130, 50, 1))]:
        with pytest.raises(ValueError, match="overlap"):
            _check_apart(x.as_strided(sizes, strides))


def test_weights_refuse_before_any_launch():
    q, cache, tree, layer, kn, _ = _args()
    with pytest.raises(ValueError, match="CUDA tensor"):
        attention_weights(q, torch.zeros(4, 3), cache, tree, layer, kn)
    with pytest.raises(ValueError, match="layer"):
        attention_weights(q, torch.zeros(4, 3), cache, tree, -1, kn)
    with pytest.raises(RuntimeError, match="CUDA"):
        heaviest(torch.zeros(2, 9), 4)


def test_retain_and_free():
    pool = _pool()
    keep = torch.zeros(1, 2, 4, dtype=torch.int32)
    src, dst = torch.arange(4, 12), torch.arange(16, 20)
    with pytest.raises(RuntimeError, match="CUDA"):
        pool.retain(src, keep, dst)
    for bad in (keep.long(), keep[:, :1], keep[..., :3]):
        with pytest.raises(ValueError, match="keep must be"):
            pool.retain(src, bad, dst)
    with pytest.raises(ValueError, match="16 bytes"):
        _pool(d=4).retain(src, keep, dst)
    slots = pool.alloc(6)
    free = pool.usage()["free"]
    pool.free(slots)
    assert pool.usage()["free"] == free + 8
    with pytest.raises(_lib.QEError, match="already free"):
        pool.free(slots)


def _owners(pool):
    """(free, evictable) tokens."""
    return pool.usage()["free"], pool.usage()["evictable"]


@pytest.mark.parametrize("page", [1, 4])
def test_free_refuses_slots_of_the_tree(page):
    pool = _pool(page=page)
    a, b = pool.alloc(8), pool.alloc(8)
    pool.insert(np.arange(100, 108), a, 0)
    before = _owners(pool)
    hit = pool.match(np.arange(100, 108))
    mixed = torch.cat([hit.indices, b])
    for bad in (a, a[:4], hit.indices, mixed):
        with pytest.raises(_lib.QEError, match="tree"):
            pool.free(bad)
    assert _owners(pool) == (before[0], 0)  # locked by the match, none of b's freed
    hit.release()
    pool.free(b)
    assert _owners(pool) == (before[0] + 8, before[1])
    rest = pool.alloc(pool.usage()["free"])  # all that is free: nothing of the tree among it
    assert not set(rest.tolist()) & set(a.tolist())
    # what eviction gave back is free once, and can be handed out and given back again
    assert pool.index.evict(8) == 8
    with pytest.raises(_lib.QEError, match="already free"):
        pool.free(a)
    again = pool.alloc(8)
    assert sorted(again.tolist()) == sorted(a.tolist())
    pool.free(again)
    pool.free(rest)
    assert _owners(pool) == (32, 0)


def test_free_after_a_split_and_a_partial_eviction():
    pool = _pool(page=4)
    a = pool.alloc(12)
    pool.insert(np.arange(12), a, 0)
    c = pool.alloc(4)
    pool.insert(np.r_[np.arange(8), 50, 51, 52, 53], torch.cat([a[:8], c]), 8)  # splits a's node
    assert pool.index.evict(4) == 4  # one of the two tails
    with pytest.raises(_lib.QEError, match="tree"):
        pool.free(a[:8])
    assert pool.index.evict(100) == 12
    with pytest.raises(_lib.QEError, match="already free"):
        pool.free(a[:8])
    assert len(set(pool.alloc(32).tolist())) == 32
    pool.clear()
    pool.free(pool.alloc(32))


@pytest.mark.parametrize("page", [1, 4])
def test_free_refuses_a_slot_twice(page):
    pool = _pool(page=page)
    a = pool.alloc(8)
    for bad in (torch.cat([a, a]), torch.cat([a, a[:1]]), torch.cat([a[4:], a[:4], a[4:]])):
        with pytest.raises(_lib.QEError, match="twice"):
            pool.free(bad)
    assert pool.usage()["free"] == 24
    pool.free(a.flip(0))  # any order
    assert len(set(pool.alloc(32).tolist())) == 32


def test_free_of_the_c_index_marks_as_it_checks():
    pool = _pool(page=1)
    a = pool.alloc(8).numpy()
    with pytest.raises(_lib.QEError, match="already free"):
        pool.index.free(np.r_[a, a[:1]])
    assert pool.usage()["free"] == 24
    pool.index.free(a)
    assert len(set(pool.alloc(32).tolist())) == 32


def test_free_takes_whole_pages_as_they_were_handed_out():
    pool = _pool(page=4)
    a, b = pool.alloc(6), pool.alloc(4)  # pages 1, 2 (two slots of it), 3
    for bad in (a[:5], a[4:5], a[5:], a[1:4], torch.cat([a[:4], b[:3]]), torch.tensor([*a[:4].tolist(), 8, 9, 10])):
        with pytest.raises(_lib.QEError, match="part of an allocated page"):
            pool.free(bad)
    for bad in (torch.tensor([0, 1, 2, 3]), torch.tensor([-4, -3]), torch.arange(36, 40)):
        with pytest.raises(_lib.QEError, match="out of range"):
            pool.free(bad)
    assert pool.usage()["free"] == 20
    pool.free(a[4:])  # its second page
    assert pool.alloc(25) is None and pool.usage()["free"] == 24
    d = pool.alloc(24)  # that page anew, whole now
    assert set(range(8, 12)) <= set(d.tolist())
    with pytest.raises(_lib.QEError, match="part of an allocated page"):
        pool.free(torch.tensor([8, 9]))
    pool.free(torch.cat([d, a[:4], b]))
    assert pool.usage()["free"] == 32
    pool.free(torch.empty(0, dtype=torch.int64))


def _batch(**over):
    base = dict(starts=16, lengths=16, tables=16, masks=0, batch=1, table_width=2, page_size=4, mask_words=0, mode=0,
                total=3, max_nodes=3, max_length=8, sum_length=8)
    base.update(over)
    return _lib.DRAFT_BATCH.pack(*base.values())


def _tree_args(batch=None, hq=4, hkv=2, d=64, dtype=1, rows=32, qt=512, scale=0.1, work=0, size=0, kd=16, q=16):
    return (batch or _batch()) + _lib.TREE_ATTENTION.pack(q, qt, 128, 16, 16, rows, kd, kd, 256, 128, 16, 512, 128, 0, work,
                                                          size, 0, hq, hkv, d, dtype, scale)


def _attend(*args, **kw):
    _lib.call("qe_tree_attention", _tree_args(*args, **kw), None)


def _weights_args(weights=16, width=11):
    return _batch() + _lib.ATTENTION_WEIGHTS.pack(16, 512, 128, 16, 32, 16, 256, 128, 16, 3, weights, 22, 11, width, 0, 4, 2,
                                                  64, 1, 0, 0.1)


@pytest.mark.parametrize("kw,match", [
    (dict(hq=3), "multiple of heads_kv"), (dict(d=96), "head_dim"), (dict(dtype=0), "dtype"), (dict(rows=30), "pool_rows"),
    (dict(qt=24), "16 bytes"), (dict(qt=64), "row of head_dim"), (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(q=24), "16-byte"), (dict(kd=8), "16-byte"), (dict(q=0), "null"),
    (dict(batch=_batch(batch=-1)), "negative"), (dict(batch=_batch(mode=3)), "mode"),
    (dict(batch=_batch(mode=1)), "masks"), (dict(batch=_batch(mode=1, masks=16, mask_words=1, max_nodes=33, total=33)), "masks"),
    (dict(batch=_batch(page_size=0)), "page_size"), (dict(batch=_batch(tables=0)), "null tables"),
    (dict(batch=_batch(starts=0)), "null starts"), (dict(batch=_batch(total=2**30)), "2\\^31"),
    (dict(batch=_batch(max_length=1 << 20, sum_length=1 << 20, table_width=1 << 18)), "workspace")])
def test_c_tree_attention_rejects(kw, match):
    with pytest.raises(ValueError, match=match):
        _attend(**kw)


@pytest.mark.parametrize("over", [dict(max_length=2**31 - 1), dict(max_nodes=2**31 - 1), dict(max_length=2**30 + 1)])
def test_c_bounds_whose_tiles_would_pass_32_bits_are_refused(over):
    """Loose bounds on the sizes of a batch are welcome, but not such that the counts of key tiles wrap round (a
    workspace of no bytes, and splits without room for their parts)."""
    batch, size = _batch(**over), ctypes.c_int64(-1)
    with pytest.raises(ValueError, match="2\\^30"):
        _lib.call("qe_tree_attention_workspace", _tree_args(batch), ctypes.byref(size))
    with pytest.raises(ValueError, match="2\\^30"):
        _attend(batch)
    with pytest.raises(ValueError, match="2\\^30"):
        _lib.call("qe_attention_weights", batch + _weights_args(width=2**33)[len(batch):], None)
    _lib.call("qe_tree_attention_workspace", _tree_args(_batch(max_length=2**30, sum_length=2**30)), ctypes.byref(size))
    assert size.value > 0


def test_c_entry_points_reject_and_accept_nothing():
    size = ctypes.c_int64(-1)
    long = _batch(max_length=1 << 20, sum_length=1 << 20)
    _lib.call("qe_tree_attention_workspace", _tree_args(long), ctypes.byref(size))
    assert size.value > 0 and size.value % 8 == 0
    with pytest.raises(ValueError):
        _lib.call("qe_tree_attention_workspace", _tree_args(hkv=3), ctypes.byref(size))
    for name in ("qe_tree_attention", "qe_attention_weights"):
        with pytest.raises(ValueError, match="null arguments"):
            _lib.call(name, None, None)
    for empty in (_batch(batch=0), _batch(total=0), _batch(max_nodes=0)):
        _attend(empty)
    with pytest.raises(ValueError, match="mask_words"):
        _lib.call("qe_tree_masks", 16, 16, 1, 40, 40, 1, 16, None, None)
    with pytest.raises(ValueError, match="width"):
        _lib.call("qe_attention_weights", _weights_args(width=10), None)
    with pytest.raises(ValueError, match="null weights"):
        _lib.call("qe_attention_weights", _weights_args(weights=0), None)
    for args in ((4, 3, 2), (4, -1, 2)):
        with pytest.raises(ValueError):
            _lib.call("qe_heaviest", 16, 1, 1, 1, 0, 0, 0, 9, None, *args, 16, None, None)
    src, dst = np.array([1, 2, 3, 4], np.int64), np.array([5, 6], np.int64)

    def retain(dst, inner=2, head=32, rows=8):
        _lib.call("qe_retain", _lib.planes(16, 0, 0, inner), rows, 1, 1, head, 16, src.ctypes.data, 4, 16, 2, 16,
                  dst.ctypes.data, None, None)

    with pytest.raises(ValueError, match="multiple of 16"):
        retain(dst, head=24)
    with pytest.raises(ValueError, match=r"\[layers, 2\]"):
        retain(dst, inner=1)
    for rows in (8, 100_000):  # marks, and sorted slots
        for bad in ([5, 5], [5, 3]):
            with pytest.raises(ValueError, match="twice, or among"):
                retain(np.array(bad, np.int64), rows=rows)
    for bad in ([5, 8], [-1, 5]):
        with pytest.raises(ValueError, match="destination slots outside"):
            retain(np.array(bad, np.int64))
    with pytest.raises(ValueError, match="source slots outside"):
        retain(np.array([0, 1], np.int64), rows=4)
