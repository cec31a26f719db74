"""Shared by the tests of the decoding and cache-eviction operators: pools with NaN outside the cached rows, and the
attention of drafted tokens in 64 bits with the error bounds its 16-bit forms keep.

Bounds. u = eps / 2 of the 16-bit type (one rounding to nearest). A kernel rounds each softmax weight to the type once
and the result once, with sums in 32 bits, so with w_j the exact weights
    |out - ref| <= u sum_j w_j |v_j| + u |ref| + 2 e sum_j w_j |v_j|
where e bounds the relative error that the 32-bit arithmetic leaves in a weight: the score's absolute error
(D + 8 additions of products summing to at most A = scale sum_d |q_d k_d|, each within 2^-23, as a matrix unit
truncates: (D + 8) 2^-23 A) and 2^-20 for the exponential and the sums. fp16 also loses weights below its smallest
step: at most 2^-25 per key, against sums of at least 1.
"""

import math

import numpy as np
import torch

from qwenedit_b200.paged import PagedKVPool


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def make_pool(layers, hkv, d, page, rooms, dtype, seed, device="cuda", spare=3, value=float("nan")):
    """A pool filled with `value` and scattered whole-page slots for requests of `rooms` tokens."""
    pages = [-(-n // page) for n in rooms]
    total = sum(pages) + spare
    budget = total * page * layers * 2 * hkv * d * torch.empty((), dtype=dtype).element_size()
    pool = PagedKVPool("test", layers, hkv, d, budget, dtype, device, page_size=page)
    pool.kv.fill_(value)
    order = np.random.default_rng(seed).permutation(np.arange(1, pool.rows // page))
    slots, at = [], 0
    for n, k in zip(rooms, pages):
        t = np.arange(n)
        mine = order[at : at + k]
        slots.append(torch.from_numpy(mine[t // page] * page + t % page).to(device))
        at += k
    return pool, slots


def fill(pool, slots, lengths, seed):
    """N(0, 1) K/V in the cached rows."""
    g = torch.Generator(device=pool.device).manual_seed(seed)
    for s, n in zip(slots, lengths):
        if n:
            v = torch.randn(pool.layers, 2, n, pool.heads, pool.head_dim, generator=g, device=pool.device)
            pool.kv[:, :, s[:n]] = v.to(pool.kv.dtype)


def chain(n):
    return torch.ones(n, n, dtype=torch.bool).tril()


def from_parents(parents):
    n = len(parents)
    see = torch.zeros(n, n, dtype=torch.bool)
    for i in range(n):
        j = i
        while j >= 0:
            see[i, j] = True
            j = parents[j]
    return see


def scores64(pool, layer, slots, length, q, kn, see, scale):
    """Of one request: scores [Hq, n, keys] in 64 bits (-inf where hidden) and A [Hq, n, keys]."""
    kc = pool.kv[layer, 0, slots[:length]].double()
    k = torch.cat([kc, kn.double()]) if kn is not None else kc
    group = q.shape[1] // pool.heads
    k = k.repeat_interleave(group, 1).permute(1, 2, 0)  # [Hq, D, keys]
    qd = q.double().transpose(0, 1)
    s = qd @ k * scale
    a = qd.abs() @ k.abs() * scale
    if kn is not None:
        hide = ~see.to(s.device)
        s[:, :, length:].masked_fill_(hide, float("-inf"))
        a[:, :, length:].masked_fill_(hide, 0.0)
    return s, a


def weight_error(a, d):
    """e of the module's text, per row."""
    top = a.amax(-1, keepdim=True) if a.shape[-1] else torch.zeros_like(a[..., :1])
    return (d + 8) * 2.0**-23 * top + 2.0**-20


def attention64(pool, layer, slots, length, q, kn, vn, see, scale):
    """Of one request: out [n, Hq, D], lse [Hq, n], and the bounds on both."""
    s, a = scores64(pool, layer, slots, length, q, kn, see, scale)
    vc = pool.kv[layer, 1, slots[:length]].double()
    v = torch.cat([vc, vn.double()]) if vn is not None else vc
    v = v.repeat_interleave(q.shape[1] // pool.heads, 1).transpose(0, 1)  # [Hq, keys, D]
    n, keys = q.shape[0], s.shape[-1]
    if keys == 0:
        zero = torch.zeros(n, q.shape[1], q.shape[2], dtype=torch.float64, device=q.device)
        none = torch.full((q.shape[1], n), float("-inf"), dtype=torch.float64, device=q.device)
        return zero, none, zero, torch.zeros_like(none)
    seen = s > float("-inf")
    w = torch.softmax(s.masked_fill(~seen.any(-1, keepdim=True), 0.0), -1) * seen
    v0 = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    out, mag = w @ v0, w @ v0.abs()
    lse = torch.logsumexp(s, -1)
    e, u = weight_error(a, q.shape[2]), half_step(q.dtype)
    tol = u * mag + u * out.abs() + 2 * e * mag
    if q.dtype == torch.float16:
        tol = tol + keys * 2.0**-25 * v0.abs().amax((1, 2))[:, None, None]
    # the sum of `keys` weights in 32 bits, the logarithm and its scaling
    lse_tol = e.squeeze(-1) + (keys + 16) * 2.0**-24 + 2.0**-21 * (1 + lse.abs().nan_to_num(posinf=0.0))
    return out.transpose(0, 1), lse, tol.transpose(0, 1), lse_tol


def weights64(s, a, lse, heads_kv, d):
    """Per key the summed weights [Hkv, keys] of one request and the bound on each (rows with lse +-inf count nothing)."""
    live = torch.isfinite(lse)
    x = s - torch.where(live, lse, torch.zeros_like(lse)).double()[..., None]
    p = torch.where(live[..., None], x.exp(), torch.zeros_like(x))
    per = (weight_error(a, d) + 2.0**-22 * torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)) * 2) * p
    hq, n, keys = p.shape
    w = p.reshape(heads_kv, hq // heads_kv * n, keys).sum(1)
    tol = per.reshape(heads_kv, hq // heads_kv * n, keys).sum(1) + w * (hq // heads_kv * n + 8) * 2.0**-24
    return w, tol + 1e-30


def default_scale(d):
    return 1.0 / math.sqrt(d)
