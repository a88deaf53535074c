"""GPU: the chunk attention (``ops.paged_chunk_attention``) with values, weights and keys of unlike and extreme
sizes, in both of its forms.

Tolerances, per output element: the bound of ``test_gpu_chunk.py``, 2^-19 A + 2^-17 S A with A = sum p |v| and
S = scale * max sum |q k| over the visible rows, bf16 2^-8 (A + |out|) more for the weights' and the result's
rounding; and what an element is held to beside its row's largest: with R = sum p * (the largest |v| of the row),
a value to 2^-29 of its row's largest element, a weight to 2^-39 of the largest of its page, 128 of them over values
that are within 2^10 of one another: 128 * 2^-39 * 2^10 + 2^-29 < 2^-21, of R.
"""

from __future__ import annotations

import importlib
import math

import numpy as np
import pytest
import torch

from test_gpu_chunk import Case, _bound, _round

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16]
FEW, MANY = [4, 2], [150, 40]  # rows of each request: the form for few rows, and the tensor cores
HEADS = {"heads": 60, "kv_heads": 60, "layers": 1, "layer": 0}  # enough of them that a CTA's run has several pages


@pytest.fixture(scope="module")
def ops():
    return importlib.import_module("unlimited-ocr-max_b200.ops")


def _np(t):
    return t.float().numpy()


def _formula(c, window=0, prefix=None):
    """The formula in float64: out, A, S and R of each row (zeros for rows in no request)."""
    q, k, v, pool = (t.double().to(DEV) for t in (c.q, c.k, c.v, c.pool[:, :, c.layer]))
    T, heads, _ = q.shape
    ref, mag, largest = (torch.zeros_like(q) for _ in range(3))
    smag = torch.zeros((T, heads), dtype=torch.float64, device=DEV)
    for b, (n, s0) in enumerate(zip(c.n, c.start)):
        if not n:
            continue
        lo, rows = int(c.offsets[b]), torch.arange(s0 + n, device=DEV)
        lut = torch.from_numpy(c.lut[b]).long().to(DEV)
        K, V = (pool[lut, i].flatten(0, 1)[: s0 + n].clone() for i in (0, 1))
        K[s0:], V[s0:] = k[lo: lo + n], v[lo: lo + n]
        K, V = (t.repeat_interleave(heads // t.shape[1], 1).permute(1, 0, 2) for t in (K, V))
        p = rows[s0:, None]
        seen = rows <= p
        if window:
            seen &= (rows > p - window) | (rows < (0 if prefix is None else int(prefix[b])))
        x = q[lo: lo + n].permute(1, 0, 2)
        K, V = K.nan_to_num(0.0, 0.0, 0.0), V.nan_to_num(0.0, 0.0, 0.0)  # hidden rows of the pool
        w = torch.softmax((x @ K.mT * c.scale).masked_fill(~seen, -math.inf), -1)
        out = lambda t: t.permute(1, 0, 2)  # noqa: E731
        ref[lo: lo + n], mag[lo: lo + n] = out(w @ V), out(w @ V.abs())
        largest[lo: lo + n] = out(w @ V.abs().amax(-1, keepdim=True))
        smag[lo: lo + n] = (x.abs() @ K.abs().mT * abs(c.scale)).masked_fill(~seen, 0).amax(-1).T
    return tuple(t.cpu().numpy() for t in (ref, mag, smag, largest))


def _check(c, ops, **more):
    """Against the formula, with the rows' largest elements in the bound (and without its absolute part)."""
    got = _np(c.run(ops, **more)[0]).astype(np.float64)
    ref, mag, smag, largest = _formula(c, **more)
    live = slice(int(c.offsets[0]), int(c.offsets[-1]))
    tol = (_bound(c.dtype, ref, mag, smag) - 1e-30 + 2.0 ** -21 * largest)[live]
    far = np.abs(got - ref)[live]
    assert (far <= tol).all(), (int((~(far <= tol)).sum()), np.argwhere(~(far <= tol))[:4].tolist(), float(np.nanmax(far / tol)))
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [FEW, MANY])
@pytest.mark.parametrize("span", [9, 12, 30, 60])
def test_rows_of_values_of_unlike_sizes(ops, oracle, dtype, n, span):
    c = Case(dtype, n, [200, 300], seed=33, **HEADS)
    rng = np.random.default_rng(span)
    for t in (c.v, c.pool[:, 1]):
        t *= torch.from_numpy(2.0 ** rng.integers(-span, span + 1, (*t.shape[:-1], 1)).astype(np.float32)).to(dtype)
    _check(c, ops)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [FEW, MANY])
def test_rows_of_zeros_among_small_and_large_ones(ops, oracle, dtype, n):
    c = Case(dtype, n, [256, 130], seed=34, **HEADS)
    rows = torch.arange(128)
    for p in range(c.pool.shape[0]):
        c.pool[p, 1][:, rows % 3 == 0] *= 0
        c.pool[p, 1][:, rows % 3 == 1] *= 2.0 ** -70
    _check(c, ops)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [FEW, MANY])
@pytest.mark.parametrize("bits", [30, 45, 60])
@pytest.mark.parametrize("first", [True, False])
def test_small_weights_of_large_values(ops, oracle, dtype, n, bits, first):
    """A page whose weights are 2^-bits of the others' and whose values 2^(bits + 10) times theirs: it makes up the
    result, whether the walk meets it first or last."""
    c = Case(dtype, n, [256, 256], seed=41, **HEADS)
    c.q += 1  # a common direction, along which the page's keys differ
    for b in (0, 1):
        page = c.lut[b, 0 if first else 1]
        c.pool[page, 0, c.layer] -= bits * math.log(2) / (c.scale * 128)
        c.pool[page, 1, c.layer] *= 2.0 ** (bits + 10)
    got = _check(c, ops)
    assert np.abs(got).max() > 2.0 ** 6


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [FEW, MANY])
@pytest.mark.parametrize("large", [1e12, 1e13, 1e30])
@pytest.mark.parametrize("whole_row", [False, True])
def test_a_large_value_of_a_later_token(ops, oracle, dtype, n, large, whole_row):
    """Tokens in front of it do not see it."""
    c = Case(dtype, n, [100, 60], seed=31, **HEADS)
    clean = _np(c.run(ops)[0])
    at = n[0] - 2  # the last row but one of the first request
    c.v[at, 1, slice(None) if whole_row else 17] = large
    got = _check(c, ops)
    # rows that do not see it: within the bound of the formula on both sides, and of the clean call
    tol = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -12
    assert (np.abs(got[:at] - clean[:at]) <= tol).all() and (got[n[0]:] == clean[n[0]:]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [FEW, MANY])
@pytest.mark.parametrize("large", [1e13, 1e30])
def test_large_values_outside_the_window(ops, oracle, dtype, n, large):
    """Rows that no token, or only the first tokens, see, on the pages of rows that all see."""
    c = Case(dtype, n, [300, 129], seed=32, **HEADS)
    for r in range(140, 180):  # behind the prefix, in front of the window of all tokens or of the later ones
        c.pool[c.lut[0, r // 128], 1, c.layer, r % 128] *= large
    _check(c, ops, window=130, prefix=[139, 0])
    _check(c, ops, window=120, prefix=[139, 0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,start", [(FEW, [400, 900]), (MANY, [400, 900])])
@pytest.mark.parametrize("size", [2.0 ** 64, 2.0 ** 66, 2.0 ** 112, 2.0 ** 120, 3e38])
@pytest.mark.parametrize("where", ["all", "first page", "last page"])
def test_values_up_to_the_largest_of_the_type(ops, oracle, dtype, n, start, size, where):
    """A mean of finite values is finite: sums of weights times values stay inside the type's range."""
    c = Case(dtype, n, start, seed=42, **HEADS)
    large = lambda t: _round((0.75 + 0.25 * torch.rand(t.shape)).numpy() * size, dtype)  # noqa: E731
    for b in (0, 1):
        for i in range(start[b] // 128):
            if where == "all" or i == (0 if where == "first page" else start[b] // 128 - 1):
                c.pool[c.lut[b, i], 1] = large(c.pool[0, 1])
    if where == "all":
        c.v = large(c.v)
    got = _check(c, ops)
    assert np.isfinite(got[: sum(n)]).all() and np.abs(got).max() > size * 2.0 ** -6


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [FEW, MANY])
@pytest.mark.parametrize("size", [1e-20, 1e-30, 1e-34])
def test_small_values(ops, dtype, n, size):
    """Results keep their bits down to 2^-126: sums of weights of at most 2^-10 times values are 2^-124 here."""
    c = Case(dtype, n, [400, 300], seed=45, **HEADS)
    c.v *= size
    c.pool[:, 1] *= size
    _check(c, ops)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [FEW, MANY])
@pytest.mark.parametrize("bad", [math.inf, -math.inf])
@pytest.mark.parametrize("factor", [1.0, -1.0])
def test_keys_with_infinite_elements(ops, oracle, dtype, n, bad, factor):
    """A row whose score is -inf has the weight 0, one whose score is +inf or NaN makes the row of out NaN: as the
    formula, whichever elements of the key are infinite, in cached and in new rows."""
    c = Case(dtype, n, [200, 130], seed=43)
    c.scale *= factor
    cached = [(0, 5, 3), (0, 150, 100), (1, 129, 0)]  # request, row, element
    for b, r, d in cached:
        c.pool[c.lut[b, r // 128], 0, c.layer, r % 128, 1, d] = bad
    c.k[1, 0, 64] = bad  # a new row; its second element of the other sign
    c.k[1, 0, 65] = -bad
    got = _np(c.run(ops)[0]).astype(np.float64)
    q, k, v, pool = (_np(t).astype(np.float64) for t in (c.q, c.k, c.v, c.pool))
    finite_nan = [0, 0]
    for b in range(2):
        for i in range(n[b]):
            t, rows = int(c.offsets[b]) + i, c.start[b] + i + 1
            for h in range(2):
                K = np.stack([pool[c.lut[b, r // 128], 0, c.layer, r % 128, h] if r < c.start[b] else k[c.offsets[b] + r - c.start[b], h]
                              for r in range(rows)])
                V = np.stack([pool[c.lut[b, r // 128], 1, c.layer, r % 128, h] if r < c.start[b] else v[c.offsets[b] + r - c.start[b], h]
                              for r in range(rows)])
                with np.errstate(invalid="ignore"):
                    s = (K * q[t, h]).sum(1) * c.scale
                if np.isnan(s).any() or (s == math.inf).any():
                    assert np.isnan(got[t, h]).all()
                    finite_nan[1] += 1
                    continue
                seen = np.isfinite(s)
                p = np.exp(s[seen] - s[seen].max())
                p /= p.sum()
                ref, mag = p @ V[seen], p @ np.abs(V[seen])
                smag = (np.abs(K[seen]) @ np.abs(q[t, h])).max() * abs(c.scale)
                tol = _bound(dtype, ref, mag, np.float64(smag)) + 2.0 ** -21 * (p @ np.abs(V[seen]).max(1))
                assert (np.abs(got[t, h] - ref) <= tol).all()
                finite_nan[0] += 1
    assert min(finite_nan) > 0


@pytest.mark.parametrize("n", [FEW, MANY])
def test_a_scale_of_zero_and_an_infinite_key(ops, n):
    """0 times an infinite score is not a number."""
    c = Case(torch.float32, n, [200, 130], seed=44)
    c.pool[c.lut[0, 0], 0, c.layer, 7, 1, 9] = math.inf
    c.scale = 0.0
    got = _np(c.run(ops)[0])
    assert np.isnan(got[: n[0], 1]).all() and np.isfinite(got[: n[0], 0]).all() and np.isfinite(got[n[0]: sum(n)]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [FEW, MANY])
@pytest.mark.parametrize("where", ["page", "window"])
def test_small_values_beside_large_ones_that_are_not_seen(ops, dtype, n, where):
    """Rows of 1e30 on the pages of rows of 1e-30: of later tokens, or outside the window."""
    c = Case(dtype, n, [300, 129], seed=46, **HEADS)
    c.v *= 1e-30
    c.pool[:, 1] *= 1e-30
    if where == "page":
        c.v[n[0] - 1] = 1e30
        c.v[sum(n) - 1] = 1e30
        _check(c, ops)
    else:
        for r in range(140, 180):
            c.pool[c.lut[0, r // 128], 1, c.layer, r % 128] *= 1e20
            c.pool[c.lut[0, r // 128], 1, c.layer, r % 128] *= 1e20
        _check(c, ops, window=120, prefix=[139, 0])
