"""GPU: a softmax warp of the chunk attention whose bounded wait runs out.

The test hook ``uocr_chunk_test_expire(mask)`` makes the softmax warps of the mask act as if their last wait of every query tile had
run out: no fault, the context stays usable. The warp stops waiting, the issuing and the copying warp learn of it and give up
in turn (the copying warp after its own 200 ms).
"""

from __future__ import annotations

import importlib

import pytest
import torch

from test_gpu_chunk import Case

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    return importlib.import_module("unlimited-ocr-max_b200.ops")


@pytest.fixture
def hook(uocr):
    lib = uocr.load()
    yield lib
    assert lib.uocr_chunk_test_expire(0) == 0


def _case(dtype):
    # 60 heads of up to 7 pages: a CTA has several query tiles
    return Case(dtype, [300, 40], [517, 100], heads=60, kv_heads=60, layers=1, layer=0, front=3, pad=5, seed=81)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("warps", [1 << 1, 1 << 6, 255])
def test_calls_after_an_expired_wait_are_correct(ops, hook, dtype, warps):
    c = _case(dtype)
    want, pool = c.run(ops)
    for _ in range(2):
        assert hook.uocr_chunk_test_expire(warps) == 0
        c.run(ops)
        assert hook.uocr_chunk_test_expire(0) == 0
        got, after = c.run(ops)
        assert torch.equal(got, want) and torch.equal(after.view(torch.uint8), pool.view(torch.uint8))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("warps", [1 << 0, 1 << 1, 1 << 6, 255])
def test_an_expired_wait_leaves_nan_and_nothing_wrong(ops, hook, dtype, warps):
    """A row's columns belong to two warps: where one of them gives up, or works on what one that gave up has left, all 128 are NaN.
    The other rows are right, and rows in no request are left."""
    c = _case(dtype)
    want, pool = c.run(ops)
    assert hook.uocr_chunk_test_expire(warps) == 0
    got, after = c.run(ops)
    assert hook.uocr_chunk_test_expire(0) == 0
    assert torch.equal(after.view(torch.uint8), pool.view(torch.uint8))
    assert torch.equal(got[:3], want[:3]) and torch.equal(got[-5:], want[-5:])
    lost = torch.isnan(got[3:-5])
    assert torch.equal(lost.any(-1), lost.all(-1))
    assert torch.equal(got[3:-5][~lost], want[3:-5][~lost])
    for w in range(8):
        if warps >> w & 1:  # rows 32 (w % 4) .. of each tile of 128
            for at, n in ((0, 300), (300, 40)):
                for r in range(at, at + n):
                    if (r - at) % 128 // 32 == w % 4:
                        assert lost[r].all()
