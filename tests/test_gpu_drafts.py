"""``drafts.tree_attention`` against attention in 64 bits over the cached and the visible drafted keys (bounds in
``tests/decode_ref.py``). Pool rows that hold no cached token are NaN, so reading one would show."""

import numpy as np
import pytest
import torch

from qwenedit_b200.drafts import DraftTree, PagedBatch, tree_attention
from tests import decode_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _case(lens, counts, hq, hkv, d, dtype, page, seed, layers=2, rooms=None):
    rooms = lens if rooms is None else rooms
    pool, slots = R.make_pool(layers, hkv, d, page, rooms, dtype, seed)
    R.fill(pool, slots, lens, seed)
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    t = sum(counts)
    rand = lambda h, x: (torch.randn(t, h, d, generator=g, device=DEV) * x).to(dtype)  # noqa: E731
    return pool, slots, rand(hq, 2.0), rand(hkv, 1.0), rand(hkv, 1.0)


def _compare(pool, slots, lens, counts, sees, q, kn, vn, out, lse, layer, scale=None):
    lo = 0
    for b, n in enumerate(counts):
        if n == 0:
            continue
        r = slice(lo, lo + n)
        ref, ref_lse, tol, lse_tol = R.attention64(
            pool, layer, slots[b], lens[b], q[r], None if kn is None else kn[r], None if vn is None else vn[r], sees[b],
            R.default_scale(q.shape[2]) if scale is None else scale)
        err = (out[r].double() - ref).abs()
        assert bool((err <= tol).all()), f"request {b}: {(err - tol).max().item()} past the bound"
        dead = ref_lse == float("-inf")
        assert torch.equal(lse[:, r] == float("-inf"), dead)
        err = torch.where(dead, torch.zeros_like(ref_lse), lse[:, r].double() - ref_lse).abs()
        assert bool((err <= lse_tol).all()), f"lse of request {b}: {(err - lse_tol).max().item()} past the bound"
        lo += n


def _random_parents(n, seed):
    rng = np.random.default_rng(seed)
    return [-1] + [int(rng.integers(max(-1, i - 6), i)) for i in range(1, n)]


HEADS = [(28, 4, 128), (8, 8, 64), (12, 1, 128), (5, 5, 128), (32, 2, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("page", [1, 6, 16, 64])
def test_one_token_each(dtype, hq, hkv, d, page):
    lens = [0, 1, 15, 16, 17, 63, 64, 65, 500, 1999]
    counts = [1] * len(lens)
    pool, slots, q, kn, vn = _case(lens, counts, hq, hkv, d, dtype, page, 1)
    out, lse = tree_attention(q, PagedBatch(pool, slots), DraftTree(counts), 1, kn, vn, return_lse=True)
    _compare(pool, slots, lens, counts, [R.chain(1)] * len(lens), q, kn, vn, out, lse, 1)
    assert pool.device_errors() == 0


@pytest.mark.parametrize("counts", [[1], [2, 0, 5, 16, 17], [31, 33], [64], [5, 130], [300]])
@pytest.mark.parametrize("kind", ["chain", "tree", "full"])
@pytest.mark.parametrize("hq,hkv,d,dtype,page", [(28, 4, 128, torch.bfloat16, 64), (6, 2, 64, torch.float16, 1),
                                                 (4, 4, 128, torch.float16, 8)])
def test_drafts(counts, kind, hq, hkv, d, dtype, page):
    lens = [97, 0, 1, 640, 33][: len(counts)]
    pool, slots, q, kn, vn = _case(lens, counts, hq, hkv, d, dtype, page, len(counts) + counts[-1])
    if kind == "tree":
        parents = [_random_parents(n, i) if n else [] for i, n in enumerate(counts)]
        tree = DraftTree(counts, sum(parents, []))
        sees = [R.from_parents(p) for p in parents]
    else:
        tree = DraftTree(counts, full=kind == "full")
        sees = [R.chain(n) if kind == "chain" else torch.ones(n, n, dtype=torch.bool) for n in counts]
    out, lse = tree_attention(q, PagedBatch(pool, slots), tree, 0, kn, vn, return_lse=True)
    _compare(pool, slots, lens, counts, sees, q, kn, vn, out, lse, 0)
    assert tree.device_errors() == 0 and pool.device_errors() == 0


@pytest.mark.parametrize("n,hq,hkv", [(1, 28, 4), (3, 28, 4), (40, 28, 4), (9, 12, 1)])
def test_long_cache_is_split_and_joined(n, hq, hkv):
    lens = [30011]
    pool, slots, q, kn, vn = _case(lens, [n], hq, hkv, 128, torch.bfloat16, 64, n, layers=1)
    out, lse = tree_attention(q, PagedBatch(pool, slots), DraftTree([n]), 0, kn, vn, return_lse=True)
    _compare(pool, slots, lens, [n], [R.chain(n)], q, kn, vn, out, lse, 0)
    again, lse2 = tree_attention(q, PagedBatch(pool, slots), DraftTree([n]), 0, kn, vn, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("length", [0, 5, 70, 4100])
@pytest.mark.parametrize("n", [6, 70])
def test_arbitrary_masks_and_rows_that_see_nothing(length, n):
    g = torch.Generator().manual_seed(n + length)
    see = torch.rand(n, n, generator=g) < 0.4
    see[2], see[:, 3] = False, False  # a row that sees no draft, a draft that no row sees
    pool, slots, q, kn, vn = _case([length], [n], 8, 2, 128, torch.bfloat16, 16, 3)
    out, lse = tree_attention(q, PagedBatch(pool, slots), DraftTree([n], visible=[see]), 0, kn, vn, return_lse=True)
    _compare(pool, slots, [length], [n], [see], q, kn, vn, out, lse, 0)
    if length == 0:
        assert not out[2].any() and bool((lse[:, 2] == float("-inf")).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("d,dtype", [(128, torch.bfloat16), (64, torch.float16)])
@pytest.mark.parametrize("n", [9, 40])
def test_hidden_drafts_with_nan_and_infinities_do_not_show(bad, d, dtype, n):
    parents = [-1] + [i // 2 - (i % 2 == 0) for i in range(1, n)]
    parents = [p if p < i else i - 1 for i, p in enumerate(parents)]
    see = R.from_parents(parents)
    pool, slots, q, kn, vn = _case([37], [n], 6, 2, d, dtype, 16, 7)
    at = n - 3
    kn_bad, vn_bad = kn.clone(), vn.clone()
    vn_bad[at, 0, 5] = bad
    vn_bad[at, 1] = bad
    kn_bad[at, 1, 3] = float("nan")
    tree = DraftTree([n], parents)
    out, lse = tree_attention(q, PagedBatch(pool, slots), tree, 0, kn_bad, vn_bad, return_lse=True)
    want, want_lse = tree_attention(q, PagedBatch(pool, slots), tree, 0, kn, vn, return_lse=True)
    clean = ~see[:, at].to(DEV)
    assert torch.equal(out[clean], want[clean]) and torch.equal(lse[:, clean], want_lse[:, clean])
    seers = see[:, at].nonzero().flatten().tolist()
    assert at in seers
    for i in seers:  # head group 0 sees one bad value of V, group 1 a NaN score
        assert not torch.isfinite(out[i, :3, 5]).any()
        assert torch.equal(out[i, :3, :5], want[i, :3, :5]) and torch.equal(out[i, :3, 6:], want[i, :3, 6:])
        assert torch.isnan(out[i, 3:]).all() and torch.isnan(lse[3:, i]).all()


@pytest.mark.parametrize("page", [2, 8, 32, 96, 128, 256])
@pytest.mark.parametrize("n", [2, 50])
def test_page_sizes(page, n):
    """Pages inside a key tile, as long as one, over several, and sizes that fit none."""
    lens = [1000, 255, 128, 5]
    pool, slots, q, kn, vn = _case(lens, [n] * 4, 8, 2, 128, torch.bfloat16, page, page + n, layers=1)
    out, lse = tree_attention(q, PagedBatch(pool, slots), DraftTree([n] * 4), 0, kn, vn, return_lse=True)
    _compare(pool, slots, lens, [n] * 4, [R.chain(n)] * 4, q, kn, vn, out, lse, 0)
    assert pool.device_errors() == 0


def test_pages_outside_the_pool_with_many_rows():
    lens, n = [700], 30
    pool, slots, q, kn, vn = _case(lens, [n], 8, 2, 128, torch.bfloat16, 64, 3, layers=1)
    cache = PagedBatch(pool, slots)
    cache.tables[0, 1] = pool.rows // 64
    cache.tables[0, 10] = -7
    out, lse = tree_attention(q, cache, DraftTree([n]), 0, kn, vn, return_lse=True)
    assert pool.device_errors() == 1
    pool.kv[:, :, slots[0][64:128]] = 0
    pool.kv[:, :, slots[0][640:]] = 0
    _compare(pool, slots, lens, [n], [R.chain(n)], q, kn, vn, out, lse, 0)


@pytest.mark.parametrize("counts,hq,hkv", [([1500], 4, 2), ([3, 2], 132, 1), ([2], 260, 2), ([1, 40], 128, 1), ([20], 127, 1)])
def test_long_drafts_and_large_groups(counts, hq, hkv):
    lens = [700, 63][: len(counts)]
    pool, slots, q, kn, vn = _case(lens, counts, hq, hkv, 64, torch.bfloat16, 16, 12, layers=1)
    out, lse = tree_attention(q, PagedBatch(pool, slots), DraftTree(counts), 0, kn, vn, return_lse=True)
    _compare(pool, slots, lens, counts, [R.chain(n) for n in counts], q, kn, vn, out, lse, 0)


@pytest.mark.parametrize("n", [1, 30])
def test_scores_that_pass_the_reference_maximum_late(n):
    """Keys whose scores jump by hundreds at the end of a tile, in its middle and tiles later."""
    pool, slots, q, kn, vn = _case([1000], [n], 8, 2, 64, torch.float16, 16, 11, layers=1)
    for at, f in ((40, 30.0), (127, 60.0), (130, 100.0), (515, 200.0), (998, 300.0)):
        pool.kv[0, 0, slots[0][at]] = (pool.kv[0, 0, slots[0][at]].float() * f).half()
    out, lse = tree_attention(q, PagedBatch(pool, slots), DraftTree([n]), 0, kn, vn, return_lse=True)
    _compare(pool, slots, [1000], [n], [R.chain(n)], q, kn, vn, out, lse, 0)


def test_scores_far_apart():
    """Maxima that grow by hundreds along the keys, and scores that vanish beside them."""
    pool, slots, q, kn, vn = _case([2000], [3], 8, 2, 64, torch.bfloat16, 16, 11)
    ramp = torch.linspace(0.1, 30.0, 2000, device=DEV)
    pool.kv[:, 0, slots[0]] = (pool.kv[:, 0, slots[0]].float() * ramp[:, None, None]).bfloat16()
    out, lse = tree_attention(q, PagedBatch(pool, slots), DraftTree([3]), 0, kn, vn, return_lse=True)
    _compare(pool, slots, [2000], [3], [R.chain(3)], q, kn, vn, out, lse, 0)


def test_cache_only_and_scale():
    lens, counts = [130, 64], [2, 3]
    pool, slots, q, _, _ = _case(lens, counts, 4, 2, 128, torch.bfloat16, 64, 5)
    out, lse = tree_attention(q, PagedBatch(pool, slots), DraftTree(counts), 0, scale=0.2, return_lse=True)
    _compare(pool, slots, lens, counts, [None, None], q, None, None, out, lse, 0, scale=0.2)


def test_lengths_below_the_slots_and_set_lengths():
    rooms, lens, counts = [200, 65, 0], [130, 1, 0], [1, 1, 1]
    pool, slots, q, kn, vn = _case(lens, counts, 28, 4, 128, torch.bfloat16, 64, 6, rooms=rooms)
    cache = PagedBatch(pool, [slots[0], slots[1], None], lens)
    tree = DraftTree(counts)
    out, lse = tree_attention(q, cache, tree, 1, kn, vn, return_lse=True)
    _compare(pool, slots, lens, counts, [R.chain(1)] * 3, q, kn, vn, out, lse, 1)
    R.fill(pool, slots, rooms, 8)
    cache.set_lengths(rooms)
    out, lse = tree_attention(q, cache, tree, 1, kn, vn, return_lse=True)
    _compare(pool, slots, rooms, counts, [R.chain(1)] * 3, q, kn, vn, out, lse, 1)
    with pytest.raises(ValueError, match="within the requests' slots"):
        cache.set_lengths([201, 1, 0])


def test_strided_inputs_and_outputs():
    """q, K and V as slices of one fused projection, out as a slice of a wider buffer."""
    lens, counts, hq, hkv, d = [70, 300], [4, 9], 8, 2, 128
    pool, slots, *_ = _case(lens, counts, hq, hkv, d, torch.bfloat16, 16, 9)
    g = torch.Generator(device=DEV).manual_seed(2)
    qkv = torch.randn(13, hq + 2 * hkv, d, generator=g, device=DEV).bfloat16()
    q, kn, vn = qkv[:, :hq], qkv[:, hq : hq + hkv], qkv[:, hq + hkv :]
    wide = torch.full((15, hq + 3, d + 8), 7.0, device=DEV).bfloat16()
    out = wide[:, 1 : hq + 1, :d]
    got, lse = tree_attention(q, PagedBatch(pool, slots), DraftTree(counts), 0, kn, vn, out=out, return_lse=True)
    assert got is out
    _compare(pool, slots, lens, counts, [R.chain(4), R.chain(9)], q, kn, vn, out, lse, 0)
    keep = torch.ones_like(wide, dtype=torch.bool)
    keep[:13, 1 : hq + 1, :d] = False
    assert bool((wide[keep] == 7.0).all())  # rows behind the last request, and everything beside the slice
    head_major = q.transpose(0, 1).contiguous().transpose(0, 1)
    got2 = tree_attention(head_major, PagedBatch(pool, slots), DraftTree(counts), 0, kn, vn)
    assert torch.equal(got2, out[:13])


def test_rows_behind_the_tree_are_not_read():
    pool, slots, q, kn, vn = _case([50], [3], 4, 2, 64, torch.bfloat16, 16, 4)
    pad = lambda t: torch.cat([t, torch.full_like(t[:2], float("nan"))])  # noqa: E731
    out = tree_attention(pad(q), PagedBatch(pool, slots), DraftTree([3]), 0, pad(kn), pad(vn))
    assert torch.equal(out[:3], tree_attention(q, PagedBatch(pool, slots), DraftTree([3]), 0, kn, vn))
    assert not out[3:].any()


def test_page_outside_the_pool_reads_zeros_and_is_reported():
    pool, slots, q, kn, vn = _case([64], [1], 4, 2, 128, torch.bfloat16, 16, 4)
    cache = PagedBatch(pool, slots)
    cache.tables[0, 2] = pool.rows // 16
    cache.tables[0, 3] = -1
    out, lse = tree_attention(q, cache, DraftTree([1]), 0, kn, vn, return_lse=True)
    assert pool.device_errors() == 1
    pool.kv[:, :, slots[0][32:]] = 0
    _compare(pool, slots, [64], [1], [R.chain(1)], q, kn, vn, out, lse, 0)


def test_device_parents_are_checked_and_rebuilt():
    n = 6
    pool, slots, q, kn, vn = _case([20], [n], 4, 2, 64, torch.bfloat16, 16, 4)
    first, second = [-1, 0, 0, 1, 2, 2], [-1, -1, 1, 2, 3, 0]
    tree = DraftTree([n], first)
    cache = PagedBatch(pool, slots)
    for parents in (first, second):
        tree.set_parents(torch.tensor(parents, dtype=torch.int32, device=DEV))
        out, lse = tree_attention(q, cache, tree, 0, kn, vn, return_lse=True)
        _compare(pool, slots, [20], [n], [R.from_parents(parents)], q, kn, vn, out, lse, 0)
    assert tree.device_errors() == 0
    tree.set_parents(torch.tensor([-1, 1, 0, 7, -2, 2], dtype=torch.int32, device=DEV))
    assert tree.device_errors() == 8 and tree.device_errors() == 0
    out, lse = tree_attention(q, cache, tree, 0, kn, vn, return_lse=True)
    _compare(pool, slots, [20], [n], [R.from_parents([-1, -1, 0, -1, -1, 2])], q, kn, vn, out, lse, 0)


def test_graphs_replay_with_new_lengths_and_keep_apart():
    """Two captured steps over one cache, replayed in turn after the cache has grown, and on another stream."""
    rooms, lens, counts = [900, 700], [130, 64], [1, 1]
    pool, slots, q, kn, vn = _case(lens, counts, 28, 4, 128, torch.bfloat16, 64, 6, rooms=rooms)
    R.fill(pool, slots, rooms, 8)
    cache, trees = PagedBatch(pool, slots, lens), [DraftTree(counts), DraftTree(counts)]
    results, graphs = [], []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for layer in (0, 1):
            tree_attention(q, cache, trees[layer], layer, kn, vn, return_lse=True)  # the library's first-use set-up
        side.synchronize()
        for layer in (0, 1):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                results.append(tree_attention(q, cache, trees[layer], layer, kn, vn, return_lse=True))
            graphs.append(g)
    torch.cuda.synchronize()
    for lengths in (lens, [900, 1], rooms):
        cache.set_lengths(lengths)
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for layer in (0, 1):
            out, lse = results[layer]
            _compare(pool, slots, lengths, counts, [R.chain(1)] * 2, q, kn, vn, out, lse, layer)


def test_host_values_are_refused_in_a_captured_graph():
    pool, slots, *_ = _case([20], [2], 4, 2, 64, torch.bfloat16, 16, 4)
    cache, tree = PagedBatch(pool, slots), DraftTree([2], [-1, 0])
    parents = torch.tensor([-1, -1], dtype=torch.int32, device=DEV)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for call in (lambda: cache.set_lengths([3]), lambda: tree.set_parents([-1, -1]), lambda: DraftTree([1])):
            with pytest.raises(RuntimeError, match="captured graph"):
                call()
        tree.set_parents(parents)  # a device tensor is fine
        cache.lengths.sub_(1)
    g.replay()
    assert cache.lengths.tolist() == [19] and tree.masks.flatten().tolist() == [1, 2]


def test_overlapping_calls_on_two_streams():
    """Calls of one cache and tree on two streams at once: each has its own workspace."""
    pool, slots, q, kn, vn = _case([30011], [3], 28, 4, 128, torch.bfloat16, 64, 6)
    cache, tree = PagedBatch(pool, slots), DraftTree([3])
    want = [tree_attention(q, cache, tree, layer, kn, vn) for layer in (0, 1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for layer, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[layer].append(tree_attention(q, cache, tree, layer, kn, vn))
    torch.cuda.synchronize()
    for layer in (0, 1):
        for out in got[layer]:
            assert torch.equal(out, want[layer])


def test_rows_past_32_bit_offsets():
    """Cached rows whose element offset passes 2^31 (a pool of 4.4 million rows of 512 elements)."""
    rows = 4_400_000
    kv = torch.empty(1, 2, rows, 4, 128, dtype=torch.bfloat16, device=DEV)
    from qwenedit_b200.paged import PagedKVPool

    pool = PagedKVPool("big", 1, 4, 128, (rows - 1) * 2 * 512 * 2, torch.bfloat16, DEV, page_size=1, kv=kv)
    slots = [torch.arange(rows - 1, rows - 400, -3, device=DEV)]
    lens = [len(slots[0])]
    R.fill(pool, slots, lens, 3)
    g = torch.Generator(device=DEV).manual_seed(5)
    q, kn, vn = (torch.randn(2, h, 128, generator=g, device=DEV).bfloat16() for h in (28, 4, 4))
    out, lse = tree_attention(q, PagedBatch(pool, slots), DraftTree([2]), 0, kn, vn, return_lse=True)
    _compare(pool, slots, lens, [2], [R.chain(2)], q, kn, vn, out, lse, 0)


def test_nothing_to_do():
    pool, slots, *_ = _case([5], [0], 4, 2, 64, torch.bfloat16, 1, 4)
    none = torch.empty(0, 4, 64, dtype=torch.bfloat16, device=DEV)
    out, lse = tree_attention(none, PagedBatch(pool, slots), DraftTree([0]), return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (4, 0)
    out = tree_attention(none, PagedBatch(pool, []), DraftTree([]))
    assert out.shape == (0, 4, 64)
