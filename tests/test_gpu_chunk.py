"""GPU: attention of a chunk of new tokens over the paged cache (``ops.paged_chunk_attention``) against
its formula in float64, fp32 and bf16.

Tolerances, per output element, from the arithmetic. Let A = sum p |v| (the size of what is summed) and
S = scale * max sum |q k| over the visible rows.
* A score sums 128 products in fp32 (or of operands held to 2^-22 of their value), in at most 32 steps,
  each off by at most 2^-23 of the partial sums: |ds| <= 2^-18 S. A weight e^(s - m) / l then is off by
  at most 2 |ds| of itself, and by 2^-20 for the exponential, its argument's rounding and its split.
* The weighted sum adds in steps of 16 rows and then of 128: 2^-20 A for up to a few thousand rows.
* bf16 rounds each weight once (2^-8 of it) and the result once (2^-8 of it).
"""

from __future__ import annotations

import importlib
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    return importlib.import_module("unlimited-ocr-max_b200.ops")


def _round(a, dtype):
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(dtype)


def _bound(dtype, ref, mag, smag):
    err = mag * (2.0 ** -19 + 2.0 ** -17 * smag[..., None])
    if dtype == torch.bfloat16:
        err = err + 2.0 ** -8 * mag + 2.0 ** -8 * np.abs(ref)
    return err + 1e-30


class Case:
    """Inputs of one call: every row of the pool that is not a cached row of some request is NaN, and so
    are the rows of q, k and v that belong to no request."""

    def __init__(self, dtype, n, start, *, heads=2, kv_heads=2, layers=2, layer=1, front=0, pad=0, seed=0, size=1.0,
                 lut_pad=0):
        rng = np.random.default_rng(seed)
        self.dtype, self.n, self.start, self.layer = dtype, list(n), list(start), layer
        B = len(self.n)
        used = [max(1, -(-(a + b) // 128)) for a, b in zip(self.n, self.start)]
        cols, pages = max(used) + lut_pad, sum(used) + 1
        perm = rng.permutation(pages - 1).astype(np.int32)
        self.lut = np.full((B, cols), pages - 1, np.int32)
        at = 0
        pool = np.full((pages, 2, layers, 128, kv_heads, 128), np.nan, np.float32)
        for b in range(B):
            self.lut[b, :used[b]] = perm[at:at + used[b]]
            at += used[b]
            for r in range(self.start[b]):
                pool[self.lut[b, r // 128], :, layer, r % 128] = rng.standard_normal((2, kv_heads, 128)) * size
        self.offsets = np.asarray([front + sum(self.n[:b]) for b in range(B + 1)], np.int32)
        T = int(self.offsets[-1]) + pad
        self.q, self.k, self.v = (np.full((T, h, 128), np.nan, np.float32) for h in (heads, kv_heads, kv_heads))
        live = slice(front, T - pad)
        for t in (self.q, self.k, self.v):
            t[live] = rng.standard_normal(t[live].shape) * size
        self.q, self.k, self.v, self.pool = (_round(t, dtype) for t in (self.q, self.k, self.v, pool))
        self.scale = 1.0 / math.sqrt(128) / size ** 2
        self.out = _round(rng.standard_normal(self.q.shape), dtype)

    def run(self, ops, **more):
        t = lambda a: (a if isinstance(a, torch.Tensor) else torch.from_numpy(np.asarray(a, np.int32))).to(DEV)  # noqa: E731
        if more.get("prefix") is not None:
            more["prefix"] = t(more["prefix"])
        pool, out = t(self.pool), t(self.out)
        got = ops.paged_chunk_attention(t(self.q), t(self.k), t(self.v), pool, self.layer, t(self.lut), t(self.offsets),
                                        t(self.start), self.scale, out=out, **more)
        assert got is out
        return out.cpu(), pool.cpu()

    def check(self, ops, oracle, **more):
        got, pool = self.run(ops, **more)
        f = lambda t: t.float().numpy()  # noqa: E731
        ref, mag, smag, after = oracle.paged_chunk_attention_ref(
            f(self.q), f(self.k), f(self.v), f(self.pool), self.layer, self.lut, self.offsets, self.start, self.scale,
            more.get("window", 0), more.get("prefix"), out=f(self.out))
        # the pool: new rows bit for bit, nothing else touched
        assert torch.equal(pool.view(torch.uint8), _round(after, self.dtype).view(torch.uint8))
        live = slice(int(self.offsets[0]), int(self.offsets[-1]))
        rest = [i for i in range(len(got)) if not live.start <= i < live.stop]
        assert torch.equal(got[rest], self.out[rest])
        far = np.abs(got.double().numpy()[live] - ref[live])
        bad = ~(far <= _bound(self.dtype, ref, mag, smag)[live])
        assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), float(np.nanmax(far)))
        return got


TYPES = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,start", [
    ([1], [0]), ([1], [1]), ([1], [127]), ([1], [128]), ([1], [639]),
    ([1] * 8, [0, 36, 299, 200, 127, 128, 511, 639]),
    ([5, 1, 0, 3], [250, 0, 40, 126]),
    ([127], [0]), ([128], [0]), ([129], [0]), ([130], [3]), ([300], [517]),
    ([2, 257, 0, 64, 31], [383, 0, 5, 129, 1000]),
])
def test_against_the_formula(ops, oracle, dtype, n, start):
    Case(dtype, n, start, seed=len(n) + sum(n)).check(ops, oracle)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (10, 10), (8, 1), (6, 2), (7, 1), (40, 8)])
def test_head_layouts(ops, oracle, dtype, heads, kv_heads):
    Case(dtype, [1, 37], [70, 150], heads=heads, kv_heads=kv_heads, layers=1, layer=0, seed=heads).check(ops, oracle)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,prefix", [
    (1, None), (1, [0, 0]), (1, [130, 1]), (128, [200, 0]), (100, None), (129, [5, 400]), (1000, [3, 3]), (64, [10**9, 256]),
    (2**31 - 1, None),
])
def test_window_and_prefix(ops, oracle, dtype, window, prefix):
    Case(dtype, [70, 200], [450, 333], seed=window % 97).check(ops, oracle, window=window, prefix=prefix)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_in_no_request_are_left(ops, oracle, dtype):
    Case(dtype, [3, 0, 140], [130, 7, 0], front=2, pad=131, seed=3, lut_pad=3).check(ops, oracle)


@pytest.mark.parametrize("size", [1e-12, 1e-3, 300.0, 1e9])
def test_fp32_values_of_any_size(ops, oracle, size):
    """The products' operands are scaled into their type's range, by powers of two."""
    Case(torch.float32, [130, 2], [5, 300], seed=11, size=size).check(ops, oracle)


def test_fp32_rows_of_unlike_sizes(ops, oracle):
    """Rows of one tile from 2^-30 to 2^30: each product to its own rows' precision for the scores; a
    value to 2^-38 of the largest value of its 128 rows, on top of the derived bound."""
    c = Case(torch.float32, [150], [200], seed=12)
    rng = np.random.default_rng(1)
    for t in (c.k, c.pool[:, 0]):
        t *= torch.from_numpy(2.0 ** rng.integers(-30, 1, (*t.shape[:-1], 1)).astype(np.float32))
    c.check(ops, oracle)


@pytest.mark.parametrize("dtype", TYPES)
def test_what_a_row_does_not_see_does_not_reach_it(ops, oracle, dtype):
    """A later token's key and value are NaN or infinite: earlier tokens of the chunk are untouched, the
    token itself and the ones behind it are not finite."""
    for bad in (math.nan, math.inf, -math.inf):
        c = Case(dtype, [150], [100], seed=21)
        clean = c.run(ops)[0]
        c.v[90, 1, 17] = bad
        got = c.run(ops)[0]
        assert torch.equal(got[:90], clean[:90]) and torch.equal(got[:, 0], clean[:, 0])
        keep = [d for d in range(128) if d != 17]
        assert not torch.isfinite(got[90:, 1, 17]).any() and torch.isfinite(got[90:, 1][:, keep]).all()
        c = Case(dtype, [150], [100], seed=21)
        c.k[90, 1] = math.nan
        got = c.run(ops)[0]
        assert torch.equal(got[:90], clean[:90]) and torch.isnan(got[90:, 1]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows_of_a_fused_projection(ops, oracle, dtype):
    c = Case(dtype, [33, 100], [64, 200], heads=4, kv_heads=2, seed=31)
    want, pool_want = c.run(ops)
    fused = torch.cat([c.q, c.k, c.v], dim=1).to(DEV)
    pool = c.pool.to(DEV)
    i32 = lambda a: torch.from_numpy(np.asarray(a, np.int32)).to(DEV)  # noqa: E731
    got = ops.paged_chunk_attention(fused[:, :4], fused[:, 4:6], fused[:, 6:], pool, 1, i32(c.lut), i32(c.offsets),
                                    i32(c.start), c.scale)
    assert torch.equal(got.cpu(), want) and torch.equal(pool.cpu().view(torch.uint8), pool_want.view(torch.uint8))
    odd = torch.empty((133, 4, 130), dtype=dtype, device=DEV)[:, :, 1:129]  # heads apart, and not on 16 bytes
    odd.copy_(fused[:, :4])
    pool = c.pool.to(DEV)
    got = ops.paged_chunk_attention(odd, fused[:, 4:6], fused[:, 6:], pool, 1, i32(c.lut), i32(c.offsets),
                                    i32(c.start), c.scale)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,start,heads,kv_heads,window,prefix", [
    ([3, 1, 2, 0], [300, 129, 640, 5], 4, 2, 0, None), ([2] * 5, [128, 127, 255, 1, 0], 2, 2, 0, None),
    ([3, 1, 2], [700, 400, 128], 2, 2, 64, [10, 0, 200]), ([1, 1], [600, 130], 8, 1, 1, None), ([4], [900], 6, 3, 130, [129]),
    ([40] + [1] * 9, [200] + [37 * i for i in range(9)], 2, 2, 0, None),  # one request of many rows among single ones
    ([9, 30, 7], [250, 100, 0], 2, 2, 40, [3, 100, 0]), ([16, 16], [300, 140], 1, 1, 0, None), ([6], [250], 2, 2, 0, None),
])
def test_few_rows(ops, oracle, dtype, n, start, heads, kv_heads, window, prefix):
    """The form for few rows a request: tiles of 1 to 8 rows, several of them where a request has more."""
    Case(dtype, n, start, heads=heads, kv_heads=kv_heads, seed=sum(n) + heads).check(ops, oracle, window=window, prefix=prefix)


@pytest.mark.parametrize("dtype", TYPES)
def test_few_rows_and_what_they_do_not_see(ops, oracle, dtype):
    """As test_what_a_row_does_not_see..., in the form for few rows: tokens in front of a key or value that is not
    finite are untouched, those behind it take it in."""
    for bad in (math.nan, math.inf):
        c = Case(dtype, [4, 1], [100, 7], seed=22)
        clean = c.run(ops)[0]
        c.v[2, 1, 17] = bad
        got = c.run(ops)[0]
        assert torch.equal(got[:2], clean[:2]) and torch.equal(got[4:], clean[4:])
        assert not torch.isfinite(got[2:4, 1, 17]).any() and torch.isfinite(got[2:4, 1, :17]).all()
        c = Case(dtype, [4, 1], [100, 7], seed=22)
        c.k[2, 1] = math.nan
        got = c.run(ops)[0]
        assert torch.equal(got[:2], clean[:2]) and torch.isnan(got[2:4, 1]).all() and torch.equal(got[:, 0], clean[:, 0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [[2, 3], [140, 20]])
@pytest.mark.parametrize("factor", [-1.0, 0.0])
def test_scales_below_and_at_zero(ops, oracle, dtype, n, factor):
    c = Case(dtype, n, [50, 129], seed=23)
    c.scale *= factor
    c.check(ops, oracle)


@pytest.mark.parametrize("dtype", TYPES)
def test_scores_that_grow_along_the_cache(ops, oracle, dtype):
    """Keys that grow from page to page, so that the maxima are raised over and over, and keys that shrink."""
    for order in (1, -1):
        c = Case(dtype, [200], [900], seed=24)
        grow = torch.linspace(0.1, 8.0, 900)[::order] if order == 1 else torch.linspace(0.1, 8.0, 900).flip(0)
        for r in range(900):
            c.pool[c.lut[0, r // 128], 0, c.layer, r % 128] *= grow[r].to(dtype)
        c.check(ops, oracle)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_requests(ops, oracle, dtype):
    rng = np.random.default_rng(5)
    for most, B in ((4, 300), (60, 70)):  # the forms for few rows and for many
        n = rng.integers(0, most, B).tolist()
        Case(dtype, n, rng.integers(0, 200, B).tolist(), heads=1, kv_heads=1, layers=1, layer=0, seed=B).check(ops, oracle)


def test_as_many_requests_as_a_call_takes(ops, oracle):
    rng = np.random.default_rng(6)
    n = rng.integers(0, 2, 8192).tolist()
    Case(torch.bfloat16, n, rng.integers(0, 12, 8192).tolist(), heads=1, kv_heads=1, layers=1, layer=0, seed=9).check(ops, oracle)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [[2, 3], [140, 20]])
def test_the_widest_window(ops, oracle, dtype, n):
    Case(dtype, n, [300, 0], seed=27).check(ops, oracle, window=2 ** 31 - 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [2, 200])
def test_pages_beyond_32_bits_of_offset(ops, dtype, n):
    """The same cache in a small pool and, page by page, at the end of one of more than 2^32 elements."""
    c = Case(dtype, [n], [300], heads=2, kv_heads=1, layers=1, layer=0, seed=28)
    args = _flat(c)
    want = ops.paged_chunk_attention(*args)
    used, pages, layers, layer = c.lut.shape[1], 530, 256, 255
    assert pages * 2 * layers * 128 * 128 > 2 ** 32
    pool = torch.empty((pages, 2, layers, 128, 1, 128), dtype=dtype, device=DEV)
    far = [pages - 2 - i for i in range(used)]
    for i, p in enumerate(far):
        pool[p, :, layer] = c.pool[c.lut[0, i], :, 0].to(DEV)
        pool[p, :, layer - 1] = 7
    lut = torch.tensor([far], dtype=torch.int32, device=DEV)
    got = ops.paged_chunk_attention(*args[:3], pool, layer, lut, *args[6:])
    assert torch.equal(got, want)
    for i, p in enumerate(far):
        assert torch.equal(pool[p, :, layer].view(torch.uint8), args[3][c.lut[0, i], :, 0].view(torch.uint8))
        assert bool((pool[p, :, layer - 1] == 7).all())
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    pool[0].zero_(), pool[1].zero_()
    ops.copy_pages(pool, i32([far[0]]), i32([0]))
    assert torch.equal(pool[0].view(torch.uint8), pool[far[0]].view(torch.uint8))
    ops.compact_rows(pool, i32([far[:1]]), i32([[1]]), i32([[3, 100]]), i32([2]))
    assert torch.equal(pool[1, :, :, :2].view(torch.uint8), pool[far[0]][:, :, [3, 100]].view(torch.uint8))
    assert bool((pool[1, :, :, 2:] == 0).all())


def test_a_table_far_wider_than_its_requests(ops, oracle):
    """Most entries name the null page; the operands of all heads at once would pass a gigabyte, so that the heads
    are taken in several passes."""
    Case(torch.float32, [150, 30], [260, 0], heads=6, kv_heads=3, seed=25, lut_pad=2500).check(ops, oracle)


def test_the_first_call_of_a_process_may_be_captured():
    import subprocess
    import sys
    from pathlib import Path

    code = """
import importlib, torch
ops = importlib.import_module("unlimited-ocr-max_b200.ops")
i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
for n, heads in ((200, 2), (2, 2)):
    pool = torch.randn(4, 2, 1, 128, heads, 128, device="cuda")
    q, k, v = (torch.randn(n, heads, 128, device="cuda") for _ in range(3))
    lut, off, start, out = i([[0, 1, 2]]), i([0, n]), i([40]), torch.zeros_like(q)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.paged_chunk_attention(q, k, v, pool, 0, lut, off, start, 0.1, out=out)
    assert not out.any()
    g.replay()
    want = ops.paged_chunk_attention(q, k, v, pool, 0, lut, off, start, 0.1)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_refusals(ops):
    c = Case(torch.float32, [5], [10], seed=26)
    q, k, v, pool, layer, lut, off, start, scale = _flat(c)
    call = lambda **m: ops.paged_chunk_attention(*({"q": q, "k": k, "v": v, "pool": pool, "layer": layer, "lut": lut, "off": off,  # noqa: E731
                                                   "start": start, "scale": scale} | m).values())
    for bad, kind in (({"q": q.bfloat16()}, TypeError), ({"k": k[:, :1]}, ValueError), ({"v": v[:3]}, ValueError), ({"lut": lut.long()}, TypeError),
                      ({"off": off[:1]}, ValueError), ({"start": start.long()}, TypeError), ({"layer": 2}, ValueError),
                      ({"pool": pool[:, :, :, :64]}, ValueError), ({"pool": pool.transpose(3, 4)}, ValueError), ({"pool": pool.half()}, TypeError),
                      ({"q": q[0]}, ValueError), ({"scale": math.inf}, ValueError), ({"k": pool[0, 0, 0, :5]}, ValueError)):
        with pytest.raises(kind):
            call(**bad)
    with pytest.raises(ValueError, match="window"):
        ops.paged_chunk_attention(q, k, v, pool, layer, lut, off, start, scale, window=-1)
    with pytest.raises(ValueError, match="overlaps q"):
        ops.paged_chunk_attention(q, k, v, pool, layer, lut, off, start, scale, out=q)
    with pytest.raises(ValueError, match="out must be"):
        ops.paged_chunk_attention(q, k, v, pool, layer, lut, off, start, scale, out=torch.empty_like(q).transpose(0, 1))


def _flat(c):
    i32 = lambda a: torch.from_numpy(np.asarray(a, np.int32)).to(DEV)  # noqa: E731
    return [c.q.to(DEV), c.k.to(DEV), c.v.to(DEV), c.pool.to(DEV), c.layer, i32(c.lut), i32(c.offsets), i32(c.start),
            c.scale]


@pytest.mark.parametrize("dtype", TYPES)
def test_repeats_bit_for_bit_and_from_other_streams(ops, dtype):
    c = Case(dtype, [300, 1, 77], [900, 640, 0], seed=41)
    args = _flat(c)
    want = ops.paged_chunk_attention(*args)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams * 3:  # at once on three streams: each call has a workspace of its own
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(ops.paged_chunk_attention(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("dtype", TYPES)
def test_two_graphs_replayed_in_turn_follow_their_inputs(ops, dtype):
    """The lengths are read on the device: a graph captured once serves chunks of other lengths."""
    c, d = Case(dtype, [130, 7], [200, 64], seed=51, pad=20), Case(dtype, [4, 150], [1, 390], seed=52, pad=3)
    graphs = []
    for x in (c, d):
        args = _flat(x)
        out = torch.zeros_like(args[0])
        ops.paged_chunk_attention(*args, out=out)
        torch.cuda.synchronize()
        out.zero_()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.paged_chunk_attention(*args, out=out)
        graphs.append((g, args, out))
    for g, _, out in graphs * 2:
        out.zero_()
        g.replay()
    torch.cuda.synchronize()
    for x, (_, args, out) in zip((c, d), graphs):
        want = ops.paged_chunk_attention(*_flat(x), out=torch.zeros_like(args[0]))
        assert torch.equal(out.view(torch.uint8), want.view(torch.uint8))
    # other lengths, the same graph: request 0 brings 100 rows, request 1 none
    g, args, out = graphs[0]
    args[6].copy_(torch.tensor([0, 100, 100], dtype=torch.int32))
    out.zero_()
    g.replay()
    again = _flat(c)
    again[6] = args[6].clone()
    want = ops.paged_chunk_attention(*again, out=torch.zeros_like(out))
    torch.cuda.synchronize()
    assert torch.equal(out.view(torch.uint8), want.view(torch.uint8))


def test_no_requests_and_no_rows(ops):
    z = lambda *s, dt=torch.float32: torch.zeros(s, dtype=dt, device=DEV)  # noqa: E731
    i = torch.int32
    pool = z(2, 2, 1, 128, 2, 128)
    assert ops.paged_chunk_attention(z(0, 2, 128), z(0, 2, 128), z(0, 2, 128), pool, 0, z(1, 1, dt=i), z(2, dt=i),
                                     z(1, dt=i), 1.0).shape == (0, 2, 128)
    out = torch.ones((3, 2, 128), device=DEV)
    ops.paged_chunk_attention(z(3, 2, 128), z(3, 2, 128), z(3, 2, 128), pool, 0, z(0, 1, dt=i), z(1, dt=i), z(0, dt=i),
                              1.0, out=out)
    ops.paged_chunk_attention(z(3, 2, 128), z(3, 2, 128), z(3, 2, 128), pool, 0, z(2, 1, dt=i), z(3, dt=i), z(2, dt=i),
                              1.0, out=out)
    assert bool((out == 1).all()) and bool((pool == 0).all())


def test_pages_and_lengths_outside_the_pool_stay_inside_it(ops, oracle):
    """Bad tables and lengths read clamped pages and store nothing outside; good requests are right."""
    c = Case(torch.float32, [4, 3, 5], [130, 40, 10], seed=61)
    args = _flat(c)
    want = ops.paged_chunk_attention(*args)
    bad = _flat(c)
    bad[5] = bad[5].clone()
    bad[5][0] = torch.tensor([-1, 10**9][: bad[5].shape[1]], dtype=torch.int32)  # request 0's pages
    bad[7] = torch.tensor([10**9, 40, -5], dtype=torch.int32, device=DEV)
    bad[3][:] = 0
    got = ops.paged_chunk_attention(*bad)
    torch.cuda.synchronize()
    again = _flat(c)
    again[3][:] = 0
    fresh = ops.paged_chunk_attention(*again)
    assert torch.equal(got[4:7], fresh[4:7]) and got.shape == want.shape


@pytest.mark.parametrize("dtype", TYPES)
def test_offsets_that_do_not_ascend_stay_inside(ops, dtype):
    """Requests that lie over one another: some result, nothing outside out and the requests' pages, and a call
    after it is right."""
    c = Case(dtype, [300, 2, 40], [10, 300, 0], seed=62)
    args = _flat(c)
    want = ops.paged_chunk_attention(*args)
    for off in ([0, 342, 0, 342], [342, 0, 300, 5], [-7, 10 ** 9, 3, 2 ** 31 - 1]):
        bad = _flat(c)
        bad[6] = torch.tensor(off, dtype=torch.int32, device=DEV)
        ops.paged_chunk_attention(*bad)
        torch.cuda.synchronize()
    assert torch.equal(ops.paged_chunk_attention(*_flat(c)), want)


def test_chunks_of_any_size_make_the_same_cache(ops):
    """A prompt fed in pieces: the pool is the same bit for bit, the outputs within the bound of the
    split's other order of summation (twice the derived one, S about 10 here: 2^-12)."""
    c = Case(torch.float32, [400], [0], seed=71)
    whole = _flat(c)
    want = ops.paged_chunk_attention(*whole)
    q, k, v, pool, layer, lut, _, _, scale = _flat(c)
    at, got = 0, []
    for n in (1, 63, 128, 200, 8):
        off = torch.tensor([0, n], dtype=torch.int32, device=DEV)
        s = torch.tensor([at], dtype=torch.int32, device=DEV)
        got.append(ops.paged_chunk_attention(q[at:at + n], k[at:at + n], v[at:at + n], pool, layer, lut, off, s, scale))
        at += n
    assert torch.equal(pool.view(torch.uint8), whole[3].view(torch.uint8))
    assert bool(((torch.cat(got) - want).abs() <= 2.0 ** -12).all())
