"""``evict.attention_weights`` against sums in 64 bits (bounds in ``tests/decode_ref.py``), ``evict.heaviest`` and
``PagedKVPool.retain`` / ``free`` against plain indexing, and the operators together, as a decoding program calls
them."""

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from qwenedit_b200.attention import PagedPrefix, paged_attention
from qwenedit_b200.drafts import DraftTree, PagedBatch, tree_attention
from qwenedit_b200.evict import attention_weights, heaviest
from qwenedit_b200.paged import PagedKVPool, cat_slots
from tests import decode_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _case(lens, counts, hq, hkv, d, dtype, page, seed, layers=2, rooms=None):
    pool, slots = R.make_pool(layers, hkv, d, page, lens if rooms is None else rooms, dtype, seed)
    R.fill(pool, slots, lens, seed)
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    t = sum(counts)
    rand = lambda h, x: (torch.randn(t, h, d, generator=g, device=DEV) * x).to(dtype)  # noqa: E731
    return pool, slots, rand(hq, 2.0), rand(hkv, 1.0)


def _lse64(pool, layer, slots, lens, counts, sees, q, kn, scale):
    """The queries' exact lse, rounded to 32 bits as an input."""
    parts, lo = [], 0
    for b, n in enumerate(counts):
        s, _ = R.scores64(pool, layer, slots[b], lens[b], q[lo : lo + n], None if kn is None else kn[lo : lo + n],
                          sees[b], scale)
        parts.append(torch.logsumexp(s, -1) if s.shape[-1] else torch.full(s.shape[:2], -float("inf"), device=DEV))
        lo += n
    return torch.cat(parts, 1).float()


def _compare(w, base, pool, layer, slots, lens, counts, sees, q, kn, lse, scale):
    lo = 0
    for b, n in enumerate(counts):
        r = slice(lo, lo + n)
        s, a = R.scores64(pool, layer, slots[b], lens[b], q[r], None if kn is None else kn[r], sees[b], scale)
        ref, tol = R.weights64(s, a, lse[:, r], pool.heads, q.shape[2])
        keys = s.shape[-1]
        ref = ref + base[b, :, :keys].double()
        tol = tol + 2.0**-24 * ref.abs()
        err = (w[b, :, :keys].double() - ref).abs()
        assert bool((err <= tol).all()), f"request {b}: {(err - tol).max().item()} past the bound"
        assert torch.equal(w[b, :, keys:], base[b, :, keys:])
        lo += n


def _run(lens, counts, hq, hkv, d, dtype, page, kind="chain", seed=0, layer=1):
    pool, slots, q, kn = _case(lens, counts, hq, hkv, d, dtype, page, seed)
    if kind == "tree":
        rng = np.random.default_rng(seed)
        parents = [[-1] + [int(rng.integers(max(-1, i - 6), i)) for i in range(1, n)] if n else [] for n in counts]
        tree, sees = DraftTree(counts, sum(parents, [])), [R.from_parents(p) for p in parents]
    else:
        tree = DraftTree(counts, full=kind == "full")
        sees = [R.chain(n) if kind == "chain" else torch.ones(n, n, dtype=torch.bool) for n in counts]
    scale = R.default_scale(d)
    lse = _lse64(pool, layer, slots, lens, counts, sees, q, kn, scale)
    cache = PagedBatch(pool, slots)
    w = attention_weights(q, lse, cache, tree, layer, kn)
    assert w.shape == (len(lens), hkv, max(lens) + max(counts))
    _compare(w, torch.zeros_like(w), pool, layer, slots, lens, counts, sees, q, kn, lse, scale)
    assert torch.equal(w, attention_weights(q, lse, cache, tree, layer, kn))
    assert pool.device_errors() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (8, 8, 64), (12, 1, 128), (32, 2, 64)])
@pytest.mark.parametrize("page", [1, 6, 64])
def test_weights_of_one_token_each(dtype, hq, hkv, d, page):
    lens = [0, 1, 15, 16, 17, 63, 64, 65, 500, 1999]
    _run(lens, [1] * len(lens), hq, hkv, d, dtype, page)


@pytest.mark.parametrize("counts", [[1], [2, 0, 5, 16, 17], [31, 33], [5, 130], [300]])
@pytest.mark.parametrize("kind", ["chain", "tree", "full"])
@pytest.mark.parametrize("hq,hkv,d,dtype,page", [(28, 4, 128, torch.bfloat16, 64), (6, 2, 64, torch.float16, 1)])
def test_weights_of_drafts(counts, kind, hq, hkv, d, dtype, page):
    lens = [97, 0, 1, 640, 33][: len(counts)]
    _run(lens, counts, hq, hkv, d, dtype, page, kind, seed=len(counts) + counts[-1], layer=0)


@pytest.mark.parametrize("n,length", [(777, 1023), (1280, 0), (130, 5000)])
@pytest.mark.parametrize("d,dtype", [(128, torch.bfloat16), (64, torch.float16)])
def test_weights_of_a_prompt(n, length, d, dtype):
    _run([length], [n], 4, 2, d, dtype, 16, seed=n)


@pytest.mark.parametrize("counts,hq,hkv", [([3, 2], 132, 1), ([2], 260, 1), ([3, 40], 100, 1), ([2], 128, 1),
                                            ([1], 64, 1), ([1, 1], 100, 1), ([1, 0], 256, 2)])
def test_weights_of_large_groups(counts, hq, hkv):
    _run([300, 17][: len(counts)], counts, hq, hkv, 64, torch.bfloat16, 16, seed=hq)


@pytest.mark.parametrize("kind", ["chain", "tree"])
@pytest.mark.parametrize("n", [33, 60])
def test_weights_either_side_of_the_kernels_border(kind, n):
    """Rows a K/V head (7 a node) around the count from which the tensor-memory kernel takes over."""
    _run([900, 0, 129], [n, 3, n - 1], 28, 4, 128, torch.bfloat16, 64, kind, seed=n)


@pytest.mark.parametrize("kind", ["chain", "tree"])
@pytest.mark.parametrize("n", [8, 9, 16, 31, 32, 33])
def test_weights_of_middle_rows_over_few_and_many_keys(kind, n):
    """The border moves with the keys: few of them (every tile finds an SM) and many, at the same rows."""
    _run([900, 0, 129], [n, 3, n - 1], 28, 4, 128, torch.float16, 64, kind, seed=n)
    _run([4100, 0, 129, 1203], [n, 3, n - 1, n], 28, 4, 128, torch.bfloat16, 16, kind, seed=n)


def test_outputs_whose_rows_overlap_are_refused():
    pool, slots, q, kn = _case([20, 9], [1, 1], 4, 2, 64, torch.bfloat16, 16, 0)
    cache, tree = PagedBatch(pool, slots), DraftTree([1, 1])
    lse = torch.zeros(4, 2, device=DEV)
    store = torch.zeros(1000, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        attention_weights(q, lse, cache, tree, 0, kn, out=store.as_strided((2, 2, 21), (24, 24, 1)))
    same = torch.zeros(1, 4, 64, dtype=torch.bfloat16, device=DEV).expand(2, 4, 64)
    with pytest.raises(ValueError, match="overlap"):
        tree_attention(q, cache, tree, 0, kn, kn, out=same)


@pytest.mark.parametrize("lens,hq,hkv,d,dtype", [([70], 28, 4, 128, torch.bfloat16), ([0, 700], 6, 2, 64, torch.float16),
                                                 ([2000, 1, 130], 256, 1, 128, torch.bfloat16)])
@pytest.mark.parametrize("draft", [False, True])
def test_weights_of_a_batch_without_new_tokens(lens, hq, hkv, d, dtype, draft):
    """Every request has finished: all weights are zero, and an accumulating call leaves them as they were."""
    pool, slots, q, kn = _case(lens, [0] * len(lens), hq, hkv, d, dtype, 16, 0)
    cache, tree = PagedBatch(pool, slots), DraftTree([0] * len(lens))
    out, lse = tree_attention(q, cache, tree, 0, kn, kn, return_lse=True)
    assert out.shape == (0, hq, d) and lse.shape == (hq, 0)
    w = attention_weights(q, lse, cache, tree, 0, kn if draft else None)
    assert w.shape == (len(lens), hkv, max(lens)) and not w.any()
    base = torch.rand(len(lens), hkv, max(lens) + 5, device=DEV)
    acc = base.clone()
    attention_weights(q, lse, cache, tree, 0, kn if draft else None, out=acc, accumulate=True)
    assert torch.equal(acc, base)
    attention_weights(q, lse, cache, tree, 0, kn if draft else None, out=acc)
    assert not acc.any()


def test_weights_accumulate_into_a_wider_buffer():
    lens, counts, rooms = [130, 40], [2, 1], [200, 64]
    pool, slots, q, kn = _case(lens, counts, 28, 4, 128, torch.bfloat16, 64, 3, rooms=rooms)
    cache, tree, sees = PagedBatch(pool, slots, lens), DraftTree(counts), [R.chain(2), R.chain(1)]
    scale = R.default_scale(128)
    lse = _lse64(pool, 0, slots, lens, counts, sees, q, kn, scale)
    store = torch.rand(2, 7, 320, device=DEV)
    acc = store[:, 1:5, 16:]
    base, before = acc.clone(), store.clone()
    got = attention_weights(q, lse, cache, tree, 0, kn, out=acc, accumulate=True)
    assert got is acc
    _compare(acc, base, pool, 0, slots, lens, counts, sees, q, kn, lse, scale)
    store[:, 1:5, 16:] = before[:, 1:5, 16:]
    assert torch.equal(store, before)  # nothing beside the slice
    attention_weights(q, lse, cache, tree, 0, kn, out=acc)
    _compare(acc, torch.zeros_like(acc), pool, 0, slots, lens, counts, sees, q, kn, lse, scale)


@pytest.mark.parametrize("n", [3, 90])
def test_weights_of_rows_taken_out_and_rows_without_keys(n):
    see = R.chain(n)
    see[1] = False
    pool, slots, q, kn = _case([0], [n], 8, 2, 128, torch.bfloat16, 16, 3)
    cache, tree = PagedBatch(pool, slots), DraftTree([n], visible=[see])
    scale = R.default_scale(128)
    lse = _lse64(pool, 0, slots, [0], [n], [see], q, kn, scale)
    assert bool((lse[:, 1] == -float("inf")).all())
    lse[:, 2] = float("inf")
    w = attention_weights(q, lse, cache, tree, 0, kn)
    _compare(w, torch.zeros_like(w), pool, 0, slots, [0], [n], [see], q, kn, lse, scale)


@pytest.mark.parametrize("n", [4, 100])
def test_weights_of_hidden_nan_keys(n):
    """A draft that no node sees may hold anything; a key's NaN reaches its own weight only."""
    see = R.chain(n)
    see[:, 2] = False
    pool, slots, q, kn = _case([30], [n], 8, 2, 128, torch.bfloat16, 16, 3)
    scale = R.default_scale(128)
    lse = _lse64(pool, 0, slots, [30], [n], [see], q, kn, scale)
    cache, tree = PagedBatch(pool, slots), DraftTree([n], visible=[see])
    want = attention_weights(q, lse, cache, tree, 0, kn)
    kn[2] = float("nan")
    assert torch.equal(attention_weights(q, lse, cache, tree, 0, kn), want)
    kn[1, 0, 0] = float("nan")
    w = attention_weights(q, lse, cache, tree, 0, kn)
    assert bool(torch.isnan(w[0, 0, 31]))
    w[0, 0, 31] = want[0, 0, 31]
    assert torch.equal(w, want)


def test_weights_follow_the_attention_of_a_prompts_tail():
    """The lse of ``paged_attention`` (the encoder's partial hit): every query's weights sum to one."""
    m, n, hq, hkv = 320, 100, 28, 4
    pool, slots, q, kn = _case([m], [n], hq, hkv, 128, torch.bfloat16, 64, 5)
    vn = torch.randn_like(kn)
    _, lse = paged_attention(q, PagedPrefix(pool, slots[0]), 1, kn, vn, causal=True, return_lse=True)
    w = attention_weights(q, lse, PagedBatch(pool, slots), DraftTree([n]), 1, kn)
    # each of the G n rows of a K/V head spreads one unit; the attention's lse is within 1e-3 (its own tests)
    assert torch.allclose(w.double().sum(-1), torch.full((1, hkv), n * hq / hkv, device=DEV, dtype=torch.float64),
                          rtol=1e-3, atol=0)


# ---- heaviest ------------------------------------------------------------------------------------------------------

def _heaviest_ref(row, n, budget, sinks, recent):
    w = np.asarray(row[:n], np.float64)
    w = np.where(np.isnan(w), -np.inf, w)
    if n <= budget:
        keep = list(range(n))
    else:
        mid = sorted(range(sinks, n - recent), key=lambda i: (-w[i], i))[: budget - sinks - recent]
        keep = sorted([*range(sinks), *mid, *range(n - recent, n)])
    return keep + [-1] * (budget - len(keep))


def _check_heaviest(weights, budget, lengths=None, sinks=0, recent=0):
    keep, kept = heaviest(weights, budget, lengths, sinks, recent)
    flat = weights.reshape(-1, weights.shape[-1]).cpu().numpy()
    lens = [weights.shape[-1]] * len(flat) if lengths is None else \
        lengths.broadcast_to(weights.shape[:-1]).reshape(-1).tolist()
    k, v = keep.reshape(-1, budget).cpu().numpy(), kept.reshape(-1, budget).cpu().numpy()
    for i, row in enumerate(flat):
        want = _heaviest_ref(row, lens[i], budget, sinks, recent)
        assert k[i].tolist() == want
        there = np.asarray(want) >= 0
        np.testing.assert_array_equal(v[i][there], row[np.asarray(want)[there]])
        assert not v[i][~there].any()


@pytest.mark.parametrize("width", [1, 2, 31, 33, 1000, 4097, 20011, 70001])
@pytest.mark.parametrize("share", [0.0, 0.1, 0.5, 0.99])
def test_heaviest(width, share):
    g = torch.Generator(device=DEV).manual_seed(width)
    w = (torch.randn(5, width, generator=g, device=DEV) * 3).exp()
    budget = max(1, int(width * share))
    _check_heaviest(w, budget)
    _check_heaviest(w, budget, sinks=min(3, budget), recent=max(0, min(budget - 3, width // 7)))


@pytest.mark.parametrize("width", [100, 5000, 66000])
def test_heaviest_ties_zeros_and_non_finite(width):
    g = torch.Generator(device=DEV).manual_seed(1)
    w = torch.randint(-2, 3, (6, width), generator=g, device=DEV).float()  # many equal weights
    w[1] = 0.0
    w[1, ::3] = -0.0
    w[2, ::2] = float("nan")
    w[3, ::5] = float("inf")
    w[3, 1::5] = -float("inf")
    w[4] = float("nan")
    w[5] = torch.where(w[5] > 0, 1e-42, -1e-42)  # below the normal range
    for budget in (1, width // 3, width - 1, width, width + 7):
        _check_heaviest(w, budget)
        _check_heaviest(w, budget, sinks=min(4, budget), recent=min(budget - min(4, budget), 9))


def test_heaviest_lengths_and_strides():
    g = torch.Generator(device=DEV).manual_seed(2)
    store = torch.rand(3, 5, 4, 700, generator=g, device=DEV)
    w = store.transpose(0, 1)[:, :, 1:, 5:600]  # [5, 3, 3, 595], layers and requests the other way round
    lengths = torch.tensor([0, 1, 64, 594, 595], dtype=torch.int32, device=DEV)[:, None, None]
    for budget, sinks, recent in ((64, 0, 0), (64, 4, 60), (64, 4, 33), (1, 0, 1), (600, 4, 100)):
        _check_heaviest(w, budget, lengths, sinks, recent)
    _check_heaviest(w[:, 0, 0, ::2], 40)
    _check_heaviest(w[0, 0, 0], 40, torch.tensor(100, dtype=torch.int32, device=DEV))
    over = torch.tensor([9999, -5], dtype=torch.int32, device=DEV)  # past the row, below zero
    keep, kept = heaviest(w[:2, 0, 0], 600, over)
    assert keep[0].tolist() == list(range(595)) + [-1] * 5
    assert bool((keep[1] == -1).all()) and not kept[1].any()


@pytest.mark.parametrize("rows,width", [(7, 8193), (70, 16385), (74, 140003), (18, 140003), (3, 300001), (75, 40000),
                                        (80, 90001), (2, 600011)])
def test_heaviest_rows_shared_by_several_blocks(rows, width):
    g = torch.Generator(device=DEV).manual_seed(width)
    w = torch.rand(rows, width, generator=g, device=DEV)
    w[0] = (w[0] * 5).floor()  # ties past every part's border
    lengths = torch.randint(0, width + 1, (rows,), generator=g, device=DEV, dtype=torch.int32)
    lengths[0], lengths[1] = width, 300
    _check_heaviest(w, 1000, lengths, 4, 31)
    _check_heaviest(w[:2], width // 3, lengths[:2], 0, 5)
    keep, _ = heaviest(w, 700, lengths, 400, 300)  # nothing left to choose
    assert keep[0].tolist() == list(range(400)) + list(range(width - 300, width))


def test_heaviest_many_rows_and_none():
    g = torch.Generator(device=DEV).manual_seed(3)
    _check_heaviest(torch.rand(300, 257, generator=g, device=DEV), 100, sinks=4, recent=16)
    keep, kept = heaviest(torch.empty(0, 10, device=DEV), 4)
    assert keep.shape == (0, 4) and kept.shape == (0, 4)
    keep, kept = heaviest(torch.empty(3, 0, device=DEV), 4)
    assert bool((keep == -1).all()) and not kept.any()
    keep, kept = heaviest(torch.rand(3, 9, device=DEV), 0)
    assert keep.shape == (3, 0)


# ---- retain --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("layers,heads,d,dtype,page,length,n", [
    (3, 4, 128, torch.bfloat16, 64, 500, 130), (1, 1, 64, torch.float16, 1, 33, 33), (2, 5, 128, torch.bfloat16, 1, 1, 1),
    (2, 3, 24, torch.bfloat16, 6, 100, 31), (2, 2, 256, torch.float32, 16, 200, 65), (28, 4, 128, torch.bfloat16, 1, 4000, 1000)])
def test_retain(layers, heads, d, dtype, page, length, n):
    pool, (src, dst) = R.make_pool(layers, heads, d, page, [length, n], dtype, 3)
    pool.kv.normal_()
    g = torch.Generator(device=DEV).manual_seed(4)
    keep = torch.rand(layers, heads, length, generator=g, device=DEV).topk(n).indices.sort().values.int()
    keep[:, :, n // 2] = keep[:, :, 0]  # the same position twice
    keep[0, 0, n - 1] = -1
    want = pool.kv.clone()
    for layer in range(layers):
        for h in range(heads):
            k = keep[layer, h].long()
            there = k >= 0
            want[layer, :, dst[there], h] = pool.kv[layer, :, src[k[there]], h]
    pool.retain(src, keep, dst)
    assert torch.equal(pool.kv, want)
    assert pool.device_errors() == 0


@pytest.mark.parametrize("d,dtype", [(8, torch.bfloat16), (4, torch.float32), (136, torch.bfloat16), (68, torch.float32),
                                     (264, torch.float16), (16, torch.bfloat16), (40, torch.float16)])
@pytest.mark.parametrize("layers,heads,length,n", [(1, 3, 60, 37), (4, 2, 2500, 1201), (28, 16, 1500, 700)])
def test_retain_of_heads_of_odd_sizes(d, dtype, layers, heads, length, n):
    """Heads of 1, 17 and 33 sixteen-byte chunks among them: a warp's last turn has chunks for half its lanes."""
    pool, (src, dst) = R.make_pool(layers, heads, d, 1, [length, n], dtype, 3)
    pool.kv.normal_()
    g = torch.Generator(device=DEV).manual_seed(4)
    keep = torch.rand(layers, heads, length, generator=g, device=DEV).topk(n).indices.sort().values.int()
    keep[:, 1, ::3] = -1
    want = pool.kv.clone()
    for layer in range(layers):
        for h in range(heads):
            k = keep[layer, h].long()
            there = k >= 0
            want[layer, :, dst[there], h] = pool.kv[layer, :, src[k[there]], h]
    pool.retain(src, keep, dst)
    assert torch.equal(pool.kv, want)
    assert pool.device_errors() == 0


def test_retain_skips_and_reports_positions_past_the_sequence():
    pool, (src, dst) = R.make_pool(1, 2, 64, 1, [10, 4], torch.bfloat16, 3)
    pool.kv.normal_()
    keep = torch.tensor([[[0, 9, 10, 3], [2**31 - 1, 1, 2, 3]]], dtype=torch.int32, device=DEV)
    want = pool.kv.clone()
    for h, i, p in ((0, 0, 0), (0, 1, 9), (0, 3, 3), (1, 1, 1), (1, 2, 2), (1, 3, 3)):
        want[0, :, dst[i], h] = pool.kv[0, :, src[p], h]
    pool.retain(src, keep, dst)
    assert torch.equal(pool.kv, want) and pool.device_errors() == 1


def test_retain_past_32_bit_offsets():
    rows = 4_400_000
    kv = torch.empty(1, 2, rows, 4, 128, dtype=torch.bfloat16, device=DEV)
    pool = PagedKVPool("big", 1, 4, 128, (rows - 1) * 2 * 512 * 2, torch.bfloat16, DEV, page_size=1, kv=kv)
    src, dst = torch.arange(rows - 1, rows - 41, -1, device=DEV), torch.arange(rows - 100, rows - 90, device=DEV)
    kv[:, :, src] = torch.randn(1, 2, 40, 4, 128, device=DEV).bfloat16()
    keep = torch.arange(0, 40, 4, dtype=torch.int32, device=DEV).broadcast_to(1, 4, 10)
    pool.retain(src, keep, dst)
    assert torch.equal(kv[:, :, dst], kv[:, :, src[::4]])


def test_slots_written_in_place_are_seen():
    """The host's copy of a slot tensor is read anew after a write: by retain's checks, batches, copies."""
    pool = PagedKVPool("written", 1, 2, 64, 16 * 16 * 2 * 2 * 64 * 2, torch.bfloat16, DEV, page_size=16)
    pool.kv.normal_()
    src, dst = pool.alloc(64), pool.alloc(32)
    keep = torch.arange(32, dtype=torch.int32, device=DEV).broadcast_to(1, 2, 32)
    pool.gather(src)
    pool.retain(src, keep, dst)
    dst[5] = src[40]
    with pytest.raises(ValueError, match="twice, or among"):
        pool.retain(src, keep, dst)
    dst[5] = dst[6]
    with pytest.raises(ValueError, match="twice, or among"):
        pool.retain(src, keep, dst)
    src.copy_(src.reshape(4, 16).flip(0).reshape(-1))
    assert torch.equal(pool.gather(src), pool.kv[:, :, src])
    assert PagedBatch(pool, [src]).tables.tolist() == [[4, 3, 2, 1]]
    new = torch.randn(1, 2, 64, 2, 64, device=DEV).bfloat16()
    src.copy_(src.roll(16))
    pool.write(src, new)
    assert torch.equal(pool.kv[:, :, src], new)


# ---- together ------------------------------------------------------------------------------------------------------

def test_decode_evict_decode():
    """Two requests decode a few tokens while the weights add up; one request's cache is cut to a third by them and
    decoding goes on over the kept tokens: the attention equals 64-bit attention over those tokens, per head."""
    layers, hq, hkv, d, page, lens = 2, 8, 2, 128, 16, [150, 70]
    steps, budget = 3, 64
    pool = PagedKVPool("decode", layers, hkv, d, 64 * page * layers * 2 * hkv * d * 2, torch.bfloat16, DEV,
                       page_size=page)
    pool.index.shuffle_free(5)
    slots = [pool.alloc(n + steps) for n in lens]
    R.fill(pool, slots, lens, 1)
    cache, tree = PagedBatch(pool, slots, lens), DraftTree([1, 1])
    acc = torch.zeros(layers, 2, hkv, cache.max_length + 1, device=DEV)
    want = torch.zeros(layers, 2, hkv, cache.max_length + 1, dtype=torch.float64, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(2)
    scale = R.default_scale(d)
    for step in range(steps):
        now = [n + step for n in lens]
        for layer in range(layers):
            q, kn, vn = (torch.randn(2, h, d, generator=g, device=DEV).bfloat16() for h in (hq, hkv, hkv))
            _, lse = tree_attention(q, cache, tree, layer, kn, vn, return_lse=True)
            attention_weights(q, lse, cache, tree, layer, kn, out=acc[layer], accumulate=True)
            for b in range(2):
                s, _ = R.scores64(pool, layer, slots[b], now[b], q[b : b + 1], kn[b : b + 1], R.chain(1), scale)
                p = torch.softmax(s, -1).view(hkv, -1, s.shape[-1]).sum(1)
                want[layer, b, :, : s.shape[-1]] += p
                pool.kv[layer, 0, slots[b][now[b]]] = kn[b]
                pool.kv[layer, 1, slots[b][now[b]]] = vn[b]
        cache.set_lengths([n + 1 for n in now])
    assert torch.allclose(acc.double(), want, rtol=1e-4, atol=1e-7)

    length = lens[0] + steps
    keep, kept = heaviest(acc[:, 0], budget, torch.tensor(length, dtype=torch.int32, device=DEV), sinks=2, recent=8)
    small = pool.alloc(budget)
    pool.retain(slots[0], keep, small)
    free = pool.usage()["free"]
    pool.free(slots[0])
    assert pool.usage()["free"] == free + -(-length // page) * page
    cache2 = PagedBatch(pool, [small, slots[1]], [budget, lens[1] + steps])
    for layer in range(layers):
        q, kn, vn = (torch.randn(2, h, d, generator=g, device=DEV).bfloat16() for h in (hq, hkv, hkv))
        out, lse = tree_attention(q, cache2, tree, layer, kn, vn, return_lse=True)
        for h in range(hkv):  # each head kept its own positions
            rows = small
            ref, ref_lse, tol, lse_tol = R.attention64(pool, layer, rows, budget, q[:1], kn[:1], vn[:1], R.chain(1), scale)
            assert bool(((out[:1].double() - ref).abs() <= tol).all())
            assert bool(((lse[:, :1].double() - ref_lse).abs() <= lse_tol).all())
            assert keep[layer, h].tolist()[:2] == [0, 1] and keep[layer, h, -1].item() == length - 1
    assert cat_slots(small, slots[1]).numel() == budget + lens[1] + steps
    assert pool.device_errors() == 0


@pytest.mark.parametrize("page,dtype", [(16, torch.bfloat16), (1, torch.float16)])
def test_attention_over_a_cut_cache_is_that_over_the_kept_tokens(page, dtype):
    """The reference takes each head's keys from a copy of the pool made before ``retain``, by ``keep``; and ``keep``
    is what the accumulated weights call for."""
    layers, hq, hkv, d, length, budget, sinks, recent = 3, 12, 3, 64, 210, 70, 2, 8
    pool, (slots, small) = R.make_pool(layers, hkv, d, page, [length, budget], dtype, 7)
    R.fill(pool, [slots], [length], 1)
    cache, tree, scale = PagedBatch(pool, [slots]), DraftTree([5]), R.default_scale(d)
    g = torch.Generator(device=DEV).manual_seed(2)
    rand = lambda n, h: torch.randn(n, h, d, generator=g, device=DEV).to(dtype)  # noqa: E731
    acc = torch.zeros(layers, 1, hkv, length, device=DEV)
    for layer in range(layers):
        q = rand(5, hq) * 2
        _, lse = tree_attention(q, cache, tree, layer, return_lse=True)
        attention_weights(q, lse, cache, tree, layer, out=acc[layer])
    keep, kept = heaviest(acc[:, 0], budget, sinks=sinks, recent=recent)
    rows = acc[:, 0].cpu().numpy()
    for layer in range(layers):
        for h in range(hkv):
            want = _heaviest_ref(rows[layer, h], length, budget, sinks, recent)
            assert keep[layer, h].tolist() == want
            np.testing.assert_array_equal(kept[layer, h].cpu().numpy(), rows[layer, h][want])
    before = pool.kv.clone()
    pool.retain(slots, keep, small)
    after, one = PagedBatch(pool, [small]), DraftTree([1])
    group = hq // hkv
    for layer in range(layers):
        q, kn, vn = rand(1, hq) * 2, rand(1, hkv), rand(1, hkv)
        out, lse = tree_attention(q, after, one, layer, kn, vn, return_lse=True)
        for h in range(hkv):
            mine = slice(h * group, (h + 1) * group)
            head = SimpleNamespace(kv=before[:, :, :, h : h + 1], heads=1)
            ref, ref_lse, tol, lse_tol = R.attention64(head, layer, slots[keep[layer, h].long()], budget, q[:, mine],
                                                       kn[:, h : h + 1], vn[:, h : h + 1], R.chain(1), scale)
            assert bool(((out[:, mine].double() - ref).abs() <= tol).all())
            assert bool(((lse[mine].double() - ref_lse).abs() <= lse_tol).all())
    assert pool.device_errors() == 0
