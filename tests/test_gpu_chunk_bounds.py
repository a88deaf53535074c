"""GPU: the chunk attention (``ops.paged_chunk_attention``) with page ids, starts and offsets that lie outside, in both of its forms:
what is read is clamped, nothing outside the requests' rows is written, and the other requests are right."""

from __future__ import annotations

import importlib

import numpy as np
import pytest
import torch

from test_gpu_chunk import Case, _bound, _flat
from test_gpu_chunk_values import _formula

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16]
FEW, MANY = [4, 3, 5], [150, 3, 140]
STARTS = [130, 40, 260]


@pytest.fixture(scope="module")
def ops():
    return importlib.import_module("unlimited-ocr-max_b200.ops")


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _bits(t):
    return t.contiguous().view(torch.uint8)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [FEW, MANY])
def test_page_ids_past_the_pool(ops, dtype, n):
    """They read the pool's last page; new rows there are attended and not stored."""
    c = Case(dtype, n, STARTS, seed=91)
    pages = c.pool.shape[0]
    c.pool[-1] = torch.from_numpy(np.random.default_rng(1).standard_normal(c.pool[-1].shape).astype(np.float32)).to(dtype)
    args = _flat(c)
    for bad in ([-1, 10 ** 9, pages, -2 ** 31], [int(c.lut[0, 0]), -1, 2 ** 31 - 1, pages]):
        args[5][0] = _i32((bad * 2)[: c.lut.shape[1]])
        pool, out = c.pool.to(DEV), c.out.to(DEV)
        ops.paged_chunk_attention(*args[:3], pool, *args[4:], out=out)
        want = c.pool.clone()
        for b in range(3):
            for i in range(n[b]):
                page, row = int(args[5][b, (STARTS[b] + i) // 128]), (STARTS[b] + i) % 128
                if 0 <= page < pages:
                    want[page, 0, 1, row], want[page, 1, 1, row] = c.k[c.offsets[b] + i], c.v[c.offsets[b] + i]
        assert torch.equal(_bits(pool.cpu()), _bits(want))
        keep = c.lut.copy()
        c.lut = np.where((lut := args[5].cpu().numpy()) < 0, pages - 1, np.minimum(lut, pages - 1))
        ref, mag, smag, largest = _formula(c)
        c.lut = keep
        far = np.abs(out.double().cpu().numpy() - ref)
        assert (far <= _bound(dtype, ref, mag, smag) + 2.0 ** -21 * largest).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [FEW, MANY])
def test_starts_outside_the_table(ops, dtype, n):
    """A request that begins behind its table has no rows, one in front of it begins at 0, one whose rows pass the table's end
    loses those that do; the request between them is right."""
    c = Case(dtype, n, STARTS, seed=92)
    c.pool[:] = 0
    room = c.lut.shape[1] * 128
    for starts in ([10 ** 9, 40, -5], [room, 40, -2 ** 31], [room - 2, 40, 2 ** 31 - 1]):
        args = _flat(c)
        args[7] = _i32(starts)
        pool, out = c.pool.to(DEV), c.out.to(DEV)
        ops.paged_chunk_attention(*args[:3], pool, *args[4:], out=out)
        begin = [min(max(s, 0), room) for s in starts]
        count = [min(a, room - s) for a, s in zip(n, begin)]
        want = c.pool.clone()
        for b in range(3):
            for i in range(count[b]):
                page, row = c.lut[b, (begin[b] + i) // 128], (begin[b] + i) % 128
                if (begin[b] + i) // 128 < -(-(n[b] + STARTS[b]) // 128):  # (behind: the null page, which several requests may write)
                    want[page, 0, 1, row], want[page, 1, 1, row] = c.k[c.offsets[b] + i], c.v[c.offsets[b] + i]
        assert torch.equal(_bits(pool.cpu())[:-1], _bits(want)[:-1])
        for b in range(3):  # rows beyond the table are left
            rest = slice(int(c.offsets[b]) + count[b], int(c.offsets[b + 1]))
            assert torch.equal(_bits(out.cpu()[rest]), _bits(c.out[rest]))
        ref, mag, smag, largest = _formula(c)
        mid = slice(int(c.offsets[1]), int(c.offsets[2]))
        far = np.abs(out.double().cpu().numpy() - ref)[mid]
        assert (far <= (_bound(dtype, ref, mag, smag) + 2.0 ** -21 * largest)[mid]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [FEW, MANY])
def test_offsets_of_any_kind_write_inside_only(ops, dtype, n):
    c = Case(dtype, n, STARTS, seed=93, lut_pad=2)
    args = _flat(c)
    T, pages = len(c.q), c.pool.shape[0]
    wide = torch.full((T + 64, *c.out.shape[1:]), 7.0, dtype=dtype, device=DEV)
    for off in ([0, T, 0, T], [T, 0, n[0], 5], [-7, 10 ** 9, 3, 2 ** 31 - 1], [5, -2 ** 31, 9, T], [-2 ** 31, 2, -2 ** 31, 2 ** 31 - 1]):
        pool = c.pool.to(DEV)
        ops.paged_chunk_attention(*args[:3], pool, args[4], args[5], _i32(off), args[7], args[8], out=wide[32: 32 + T])
        assert bool((wide[:32] == 7).all()) and bool((wide[32 + T:] == 7).all())
        assert torch.equal(_bits(pool[:, :, 0].cpu()), _bits(c.pool[:, :, 0]))  # the other layer
        for b in range(3):  # cached rows are read only
            for r in range(0, STARTS[b], 13):
                at = (int(c.lut[b, r // 128]), slice(None), 1, r % 128)
                assert torch.equal(_bits(pool[at].cpu()), _bits(c.pool[at]))
        want = ops.paged_chunk_attention(*_flat(c))
        got = ops.paged_chunk_attention(*_flat(c))
        assert torch.equal(got, want) and bool(torch.isfinite(got).all())
    assert pages > 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [[1], [3], [150]])
def test_tables_rows_and_pools_of_other_layouts(ops, dtype, n):
    """Tables of uint32, transposed or cut from wider ones; broadcast keys and values; rows of one token with a stride of their own;
    a pool inside a larger tensor."""
    c = Case(dtype, n, [300], heads=4, kv_heads=2, seed=94, lut_pad=1)
    args = _flat(c)
    want = ops.paged_chunk_attention(*args)
    stored = args[3].clone()

    def same(**change):
        a = _flat(c)
        for i, v in change.items():
            a[int(i[1:])] = v
        got = ops.paged_chunk_attention(*a)
        assert torch.equal(got, want) and torch.equal(_bits(a[3]), _bits(stored))

    lut = args[5]
    same(_5=lut.to(torch.int64).to(torch.uint32))
    same(_5=lut.t().contiguous().t())
    same(_5=torch.cat([lut, lut], 1)[:, : lut.shape[1]])
    same(_5=torch.cat([lut, lut], 1).to(torch.int64).to(torch.uint32)[:, : lut.shape[1]])
    same(_6=torch.stack([args[6], args[6]], 1)[:, 0], _7=torch.stack([args[7], args[7]], 1)[:, 1])
    same(_0=torch.cat([args[0], args[0]], 1)[:, :4], _2=torch.cat([args[2], args[2], args[2]], 1)[:, 2:4])
    big = torch.zeros(c.pool.numel() + 64, dtype=dtype, device=DEV)
    pool = big[64:].view(c.pool.shape)
    pool.copy_(c.pool)
    same(_3=pool)
    assert bool((big[:64] == 0).all())
    a = _flat(c)
    one = a[1][:1, :1].expand(len(c.k), 2, 128)  # one key for all rows and heads
    a[1] = one
    b = _flat(c)
    b[1] = one.contiguous()
    assert torch.equal(ops.paged_chunk_attention(*a), ops.paged_chunk_attention(*b)) and torch.equal(_bits(a[3]), _bits(b[3]))
    with pytest.raises(ValueError, match="16-byte"):
        at = torch.zeros(c.pool.numel() + 1, dtype=dtype, device=DEV)[1:].view(c.pool.shape)
        ops.paged_chunk_attention(*args[:3], at, *args[4:])
