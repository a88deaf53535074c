"""GPU: page copies and row compaction (``ops.copy_pages``, ``ops.compact_rows``): every byte of the pool
against a plain restatement, and ``PagePool`` with the chunk and decode attention together."""

from __future__ import annotations

import importlib
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    return importlib.import_module("unlimited-ocr-max_b200.ops")


def _pool(pages, layers, heads, dtype, seed):
    bits = torch.randint(-2**31, 2**31, (pages, 2, layers, 128, heads, 128 * dtype.itemsize // 4), dtype=torch.int32,
                         generator=torch.Generator().manual_seed(seed))
    return bits.view(dtype)  # every bit pattern, NaN among them


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _same(a, b):
    return torch.equal(a.cpu().contiguous().view(torch.uint8), b.cpu().contiguous().view(torch.uint8))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pages,layers,heads,pairs,rows", [
    (3, 1, 1, [(0, 2)], None), (9, 12, 10, [(3, 8), (5, 0)], None), (9, 2, 10, [(3, 8), (3, 1), (5, 0)], [1, 127, 128]),
    (5, 3, 7, [(4, 0), (2, 1)], [0, 77]), (4, 1, 2, [(1, 1), (0, 3)], [5, 200]), (4, 1, 3, [(-1, 2), (0, 4), (7, 1), (2, 3)], None),
])
def test_copy_pages(ops, dtype, pages, layers, heads, pairs, rows):
    pool = _pool(pages, layers, heads, dtype, pages)
    want = pool.clone()
    for i, (a, b) in enumerate(pairs):
        n = 128 if rows is None else min(rows[i], 128)
        if 0 <= a < pages and 0 <= b < pages:
            want[b, :, :, :n] = pool[a, :, :, :n]
    got = pool.to(DEV)
    ops.copy_pages(got, _i32([a for a, _ in pairs]), _i32([b for _, b in pairs]), rows=None if rows is None else _i32(rows))
    assert _same(got, want)


def _compact_ref(pool, src, dst, keep, keep_len):
    old, new = pool.clone(), pool.clone()
    for b, n in enumerate(keep_len):
        for i in range(min(max(n, 0), len(keep[b]))):
            k = keep[b][i]
            if not (0 <= k < 128 * len(src[b]) and i < 128 * len(dst[b])):
                continue
            a, z = src[b][k // 128], dst[b][i // 128]
            if 0 <= a < len(pool) and 0 <= z < len(pool):
                new[z, :, :, i % 128] = old[a, :, :, k % 128]
    return new


def _kept(rng, rows, count):
    return sorted(rng.choice(rows, count, replace=False).tolist())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layers,heads", [(1, 1), (3, 10), (2, 3)])
@pytest.mark.parametrize("in_place", [True, False])
def test_compact_rows(ops, dtype, layers, heads, in_place):
    rng = np.random.default_rng(layers * 10 + heads)
    lens, counts = [640, 129, 1, 300, 500], [401, 128, 1, 0, 499]
    lists = [_kept(rng, a, b) for a, b in zip(lens, counts)]
    lists[0][:200] = list(range(200))  # a prefix that stays
    lists[0] = sorted(set(lists[0]))
    B, cols = len(lens), 5
    perm = rng.permutation(2 * B * cols).astype(int)
    src = perm[:B * cols].reshape(B, cols).tolist()
    dst = src if in_place else perm[B * cols:].reshape(B, cols)[:, :4].tolist()
    most = max(map(len, lists)) + 3
    keep = [k + [10**6] * (most - len(k)) for k in lists]
    n = [len(k) for k in lists]
    pool = _pool(2 * B * cols, layers, heads, dtype, 5)
    want = _compact_ref(pool, src, dst, keep, n)
    got = pool.to(DEV)
    ops.compact_rows(got, _i32(src), _i32(dst), _i32(keep), _i32(n))
    assert _same(got, want)


@pytest.mark.parametrize("dtype", TYPES)
def test_compact_one_long_request_in_place_and_over_shared_pages(ops, dtype):
    """Every shift is exercised: thousands of rows move down by one to many rows, tile by tile; then the
    first pages of both tables are the same and the others fresh."""
    rng = np.random.default_rng(8)
    rows, cols = 3500, 28
    kept = _kept(rng, rows, 2900)
    kept[:130] = range(130)
    kept = sorted(set(kept))
    perm = rng.permutation(60).tolist()
    src = [perm[:cols]]
    pool = _pool(60, 1, 2, dtype, 9)
    for dst in (src, [src[0][:1] + perm[cols:2 * cols - 1]]):
        want = _compact_ref(pool, src, dst, [kept], [len(kept)])
        got = pool.to(DEV)
        ops.compact_rows(got, _i32(src), _i32(dst), _i32([kept]), _i32([len(kept)]))
        assert _same(got, want)


def test_compact_rows_outside_the_tables_are_skipped(ops):
    pool = _pool(6, 1, 2, torch.float32, 3)
    src, dst, keep, n = [[0, -1], [1, 99]], [[4], [5]], [[-3, 5, 130, 300], [2, 3, 129, 200]], [4, 9]
    want = _compact_ref(pool, src, dst, keep, n)
    got = pool.to(DEV)
    ops.compact_rows(got, _i32(src), _i32(dst), _i32(keep), _i32(n))
    assert _same(got, want)


def test_nothing_to_move(ops):
    pool = _pool(2, 1, 1, torch.float32, 1).to(DEV)
    want = pool.clone()
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    ops.copy_pages(pool, none, none)
    ops.compact_rows(pool, _i32([[0]]), _i32([[1]]), torch.empty((1, 0), dtype=torch.int32, device=DEV), _i32([0]))
    assert _same(pool, want)


def test_moves_captured_in_a_graph(ops):
    pool = _pool(4, 2, 2, torch.float32, 2)
    got = pool.to(DEV)
    a, b, lut, keep, n = _i32([0]), _i32([1]), _i32([[2]]), _i32([[3, 4, 9]]), _i32([3])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.copy_pages(got, a, b)
        ops.compact_rows(got, lut, lut, keep, n)
    assert _same(got, pool)
    g.replay()
    want = pool.clone()
    want[1] = pool[0]
    assert _same(got, _compact_ref(want, [[2]], [[2]], [[3, 4, 9]], [3]))


@pytest.mark.parametrize("dtype", TYPES)
def test_a_served_prompt_forked_windowed_and_decoded(ops, dtype):
    """The operators together, as a server uses them: two prompts share one pool, one is forked after
    its prompt, all three grow by chunks and single tokens, one is cut to its prompt and its last rows,
    the pool is defragmented; every step's attention against the float64 formula over a plain host
    copy of each request's rows. Bounds as derived beside the chunk attention's tests."""
    kvp = importlib.import_module("unlimited-ocr-max_b200.kv_pages")
    heads, layers, scale = 4, 2, 1 / math.sqrt(128)
    pool = kvp.PagePool(24, layers, heads, dtype=dtype, device=DEV)
    rng = np.random.default_rng(4)
    told = {}  # request -> [rows, 2, heads, 128] of each layer, in float64

    def step(requests, counts):
        first = [pool.extend(r, c) for r, c in zip(requests, counts)]
        T = sum(counts)
        off = _i32(np.concatenate([[0], np.cumsum(counts)]).tolist())
        lut = pool.lut(requests)
        for layer in range(layers):
            q, k, v = (torch.from_numpy(rng.standard_normal((T, heads, 128)).astype(np.float32)).to(dtype) for _ in range(3))
            one = dtype == torch.float32 and max(counts) == 1 and min(counts) == 1
            if one:  # the decode step's own operator over the same pool
                got = ops.paged_decode_attention(q.to(DEV), k.to(DEV), v.to(DEV), pool.pool, layer, lut, _i32(first),
                                                 _i32([f + 1 for f in first]), scale)
            else:
                got = ops.paged_chunk_attention(q.to(DEV), k.to(DEV), v.to(DEV), pool.pool, layer, lut, off, _i32(first), scale)
            at = 0
            for r, c in zip(requests, counts):
                rows = told.setdefault(r, [np.zeros((0, 2, heads, 128))] * layers)
                rows[layer] = np.concatenate([rows[layer], np.stack([k[at:at + c].double().numpy(), v[at:at + c].double().numpy()], 1)])
                K, V = rows[layer][:, 0], rows[layer][:, 1]
                for i in range(c):
                    n = len(K) - c + i + 1
                    x = q[at + i].double().numpy()
                    s = np.einsum("hd,rhd->hr", x, K[:n]) * scale
                    p = np.exp(s - s.max(1, keepdims=True))
                    p /= p.sum(1, keepdims=True)
                    ref, mag = np.einsum("hr,rhd->hd", p, V[:n]), np.einsum("hr,rhd->hd", p, np.abs(V[:n]))
                    smag = np.einsum("hd,rhd->hr", np.abs(x), np.abs(K[:n])).max(1) * scale
                    tol = mag * (2.0 ** -19 + 2.0 ** -17 * smag[:, None])
                    if dtype == torch.bfloat16:
                        tol += 2.0 ** -8 * (mag + np.abs(ref))
                    assert (np.abs(got[at + i].double().cpu().numpy() - ref) <= tol).all()
                at += c

    pool.add("a")
    pool.add("b")
    step(["a", "b"], [300, 45])
    pool.fork("a", "c")
    told["c"] = list(told["a"])
    assert pool.table("c")[:2] == pool.table("a")[:2] and pool.table("c")[2] != pool.table("a")[2]
    step(["a", "b", "c"], [1, 1, 1])
    step(["c", "a"], [100, 7])
    kept = list(range(130)) + list(range(250, 308))
    pool.keep("a", kept)  # pages 0 and 1 are shared with c: page 1 changes, page 0 does not
    told["a"] = [t[kept] for t in told["a"]]
    step(["a", "c", "b"], [1, 1, 1])
    step(["a", "c", "b"], [70, 2, 130])
    pool.free("b")
    assert pool.defragment() == pool.pages - pool.free_pages
    step(["c", "a"], [3, 1])
    pool.keep("c", list(range(0, pool.rows("c"), 2)))
    told["c"] = [t[::2] for t in told["c"]]
    step(["a", "c"], [1, 1])
    for r in ("a", "c"):
        pool.free(r)
    assert pool.free_pages == 24
