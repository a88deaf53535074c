"""Host: what the page-pool operators refuse, before anything is launched, and the page bookkeeping of
``PagePool`` with the moves on the GPU replaced by the same moves on a host tensor."""

from __future__ import annotations

import ctypes
import importlib

import pytest
import torch

F = ctypes.c_float


@pytest.fixture()
def kvp():
    return importlib.import_module("unlimited-ocr-max_b200.kv_pages")


def _chunk(lib, **v):
    d = {"q_ld": 512, "k_ld": 256, "v_ld": 256, "T": 4, "heads": 4, "kv": 2, "dim": 128, "dtype": 0, "pages": 4,
         "layers": 2, "layer": 1, "cols": 3, "B": 2, "scale": 0.1, "window": 0, **v}
    rc = lib.uocr_paged_chunk_attention(None, d["q_ld"], None, d["k_ld"], None, d["v_ld"], d["T"], d["heads"], d["kv"],
                                        d["dim"], d["dtype"], None, d["pages"], d["layers"], d["layer"], None, d["cols"],
                                        None, None, d["B"], F(d["scale"]), d["window"], None, None, None, 0, None)
    return rc, lib.uocr_last_error().decode()


@pytest.mark.parametrize("change,code,word", [
    ({"dim": 64}, 4, "head_dim 64"), ({"dtype": 7}, 1, "dtype 7"), ({"heads": 5}, 1, "5 heads over 2"),
    ({"heads": 0}, 1, "0 heads"), ({"kv": 0}, 1, "KV heads"), ({"T": -1}, 1, "bad T"), ({"B": -1}, 1, "B -1"),
    ({"T": 1 << 40}, 1, "bad T"), ({"layer": 2}, 1, "bad pool"), ({"layer": -1}, 1, "bad pool"), ({"pages": 0}, 1, "bad pool"),
    ({"cols": 0}, 1, "bad pool"), ({"window": -1}, 1, "window -1"), ({"q_ld": 511}, 1, "row strides"),
    ({"q_ld": 514}, 1, "row strides"), ({"k_ld": 128}, 1, "row strides"), ({"dtype": 1, "v_ld": 260}, 1, "row strides"),
    ({"scale": float("nan")}, 1, "scale"), ({"scale": float("inf")}, 1, "scale"), ({}, 1, "null pointer"),
    ({"T": 0}, 0, ""), ({"B": 0}, 0, ""),
    ({"B": 8193}, 4, "8193 requests"), ({"B": 8192, "cols": 1 << 18}, 4, "tables of 8192"),
    ({"B": 64, "cols": 1 << 22, "heads": 1024, "kv": 1024, "q_ld": 1 << 17, "k_ld": 1 << 17, "v_ld": 1 << 17}, 4, "too much"),
    ({"B": 64, "cols": 1 << 13, "heads": 1024, "kv": 1024, "q_ld": 1 << 17, "k_ld": 1 << 17, "v_ld": 1 << 17}, 1, "null pointer"),
    ({"T": 1 << 28, "cols": 1 << 22}, 4, "too much"), ({"window": 1 << 31}, 1, "window"), ({"cols": (1 << 22) + 1}, 1, "bad pool"),
])
def test_chunk_attention_refusals(uocr, change, code, word):
    rc, err = _chunk(uocr.load(), **change)
    assert rc == code and word in err


def test_page_moves_refuse(uocr):
    lib = uocr.load()
    err = lambda: lib.uocr_last_error().decode()  # noqa: E731
    assert lib.uocr_copy_pages(None, 4, 1, 512, None, None, None, 1, None) == 1 and "null" in err()
    assert lib.uocr_copy_pages(None, 0, 1, 512, None, None, None, 1, None) == 1 and "bad pool" in err()
    assert lib.uocr_copy_pages(None, 4, 1, 520, None, None, None, 1, None) == 1 and "row_bytes 520" in err()
    assert lib.uocr_copy_pages(None, 4, 1, 512, None, None, None, -1, None) == 1 and "bad n" in err()
    assert lib.uocr_copy_pages(None, 4, 1, 512, None, None, None, 0, None) == 0
    assert lib.uocr_compact_rows(None, 4, 1, 512, None, 1, None, 1, None, 5, None, 1, None) == 1 and "null" in err()
    assert lib.uocr_compact_rows(None, 4, 1, 512, None, 0, None, 1, None, 5, None, 1, None) == 1 and "bad shape" in err()
    assert lib.uocr_compact_rows(None, 4, 0, 512, None, 1, None, 1, None, 5, None, 1, None) == 1 and "bad pool" in err()
    assert lib.uocr_compact_rows(None, 4, 1, 512, None, 1, None, 1, None, 0, None, 1, None) == 0


def test_host_tensors_are_refused(uocr):
    z = torch.zeros
    i = lambda *s: z(s, dtype=torch.int32)  # noqa: E731
    pool = z(2, 2, 1, 128, 2, 128)
    with pytest.raises(ValueError, match="CUDA tensor"):
        uocr.ops.paged_chunk_attention(z(1, 2, 128), z(1, 2, 128), z(1, 2, 128), pool, 0, i(1, 1), i(2), i(1), 1.0)
    with pytest.raises(ValueError, match="CUDA tensor"):
        uocr.ops.copy_pages(pool, i(1), i(1))
    with pytest.raises(ValueError, match="CUDA tensor"):
        uocr.ops.compact_rows(pool, i(1, 1), i(1, 1), i(1, 1), i(1))


class _HostMoves:
    """The two moves on a host tensor, refusing what the operators' contracts leave undefined."""

    @staticmethod
    def copy_pages(pool, src, dst, *, rows=None):
        src, dst = src.tolist(), dst.tolist()
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        for i, (a, b) in enumerate(zip(src, dst)):
            n = 128 if rows is None else int(rows[i])
            pool[b, :, :, :n] = pool[a, :, :, :n]

    @staticmethod
    def compact_rows(pool, src_lut, dst_lut, keep, keep_len):
        old = pool.clone()
        for b, n in enumerate(keep_len.tolist()):
            src, dst, rows = src_lut[b].tolist(), dst_lut[b].tolist(), keep[b].tolist()[:n]
            assert all(y > x for x, y in zip(rows, rows[1:]))
            for c, p in enumerate(dst):
                assert p not in src or src.index(p) == c
            for i, k in enumerate(rows):
                pool[dst[i // 128], :, :, i % 128] = old[src[k // 128], :, :, k % 128]


@pytest.fixture()
def pool(kvp, monkeypatch):
    monkeypatch.setattr(kvp, "ops", _HostMoves)
    return kvp.PagePool(12, 1, 1, device="cpu")


def _fill(pool, request, start, rows):
    for r in range(start, start + rows):
        page = pool.table(request)[r // 128]
        pool.pool[page, :, :, r % 128] = hash((request, r)) % 1000003


def _read(pool, request):
    t = pool.table(request)
    return [float(pool.pool[t[r // 128], 0, 0, r % 128, 0, 0]) for r in range(pool.rows(request))]


def test_requests_come_grow_fork_and_go(pool):
    pool.add("a")
    assert pool.extend("a", 200) == 0 and pool.extend("a", 60) == 200
    _fill(pool, "a", 0, 260)
    was = _read(pool, "a")
    assert pool.table("a") == [0, 1, 2] and pool.free_pages == 9
    pool.fork("a", "b")
    assert pool.table("b") == [0, 1, 3] and _read(pool, "b") == was
    pool.extend("b", 1)
    _fill(pool, "b", 260, 1)
    assert _read(pool, "a") == was  # b's new row is on its own page
    pool.free("a")
    assert pool.free_pages == 9 and _read(pool, "b")[:260] == was
    assert pool.lut(["b"]).tolist() == [[0, 1, 3]] and pool.lut(["b"], 5).tolist() == [[0, 1, 3, 12, 12]]
    pool.free("b")
    assert pool.free_pages == 12
    with pytest.raises(KeyError):
        pool.rows("b")


def test_a_fork_at_a_page_border_copies_nothing(pool):
    pool.add("a", 256)
    pool.fork("a", "b")
    assert pool.table("a") == pool.table("b") and pool.free_pages == 10
    pool.extend("b", 1)
    assert pool.table("b")[2] not in pool.table("a")


def test_shared_pages_are_copied_before_they_are_written(pool):
    pool.add("a", 256)
    _fill(pool, "a", 0, 256)
    pool.fork("a", "b")
    pool.make_writable("b", 130)
    assert pool.table("b")[0] == pool.table("a")[0] and pool.table("b")[1] != pool.table("a")[1]
    assert _read(pool, "a") == _read(pool, "b")


@pytest.mark.parametrize("forked", [False, True])
@pytest.mark.parametrize("kept", [[], [0], list(range(300)), list(range(130)) + list(range(200, 300)), list(range(1, 300, 2)),
                                  list(range(170, 300)), list(range(129)) + [299]])
def test_kept_rows(pool, forked, kept):
    pool.add("a", 300)
    _fill(pool, "a", 0, 300)
    was = _read(pool, "a")
    if forked:
        pool.fork("a", "b")
    pool.keep("a", kept)
    assert _read(pool, "a") == [was[r] for r in kept] and len(pool.table("a")) == -(-len(kept) // 128)
    if forked:
        assert _read(pool, "b") == was
        pool.free("b")
    pool.free("a")
    assert pool.free_pages == 12


def test_defragmented(pool):
    for r in "abcd":
        pool.add(r, 256)
        _fill(pool, r, 0, 256)
    pool.fork("d", "e")
    was = {r: _read(pool, r) for r in "bde"}
    pool.free("a")
    pool.free("c")
    assert pool.defragment() == 4 and pool.free_pages == 8
    assert {r: _read(pool, r) for r in "bde"} == was and sorted(pool.table("b") + pool.table("d")) == [0, 1, 2, 3]
    pool.add("f", 128)
    assert pool.table("f") == [4]


def test_a_full_pool_changes_nothing(pool, kvp):
    pool.add("a", 11 * 128)
    with pytest.raises(kvp.PoolFullError):
        pool.add("b", 300)
    with pytest.raises(kvp.PoolFullError):
        pool.extend("a", 129)
    assert pool.rows("a") == 11 * 128 and pool.free_pages == 1
    pool.extend("a", 10)
    with pytest.raises(kvp.PoolFullError):
        pool.fork("a", "c")
    with pytest.raises(KeyError):
        pool.table("c")
    with pytest.raises(ValueError):
        pool.add("a")
    with pytest.raises(ValueError):
        pool.keep("a", [3, 3])
    with pytest.raises(ValueError):
        pool.keep("a", [0, 5000])
    with pytest.raises(ValueError):
        kvp.PagePool(0, 1, 1, device="cpu")
    with pytest.raises(TypeError):
        kvp.PagePool(1, 1, 1, dtype=torch.float16, device="cpu")


@pytest.mark.parametrize("sizes", [(0, 4, 2, 0, 3, 2), (4, 4, 2, 0, 3, 0), (4, 5, 2, 0, 3, 2), (4, 0, 2, 0, 3, 2), (4, 4, 2, 7, 3, 2), (4, 4, 2, 0, 0, 2),
                                   (4, 2048, 2, 0, 3, 2), (1 << 40, 4, 2, 0, 3, 2), (4, 4, 2, 0, 3, 8193), (4, 4, 2, 0, (1 << 22) + 1, 2),
                                   (4, 4, 2, 0, 1 << 18, 8192), (4, 1024, 1024, 0, 1 << 22, 64), (1 << 28, 4, 2, 0, 1 << 22, 2)])
def test_no_workspace_for_sizes_that_the_call_refuses(uocr, sizes):
    lib = uocr.load()
    T, heads, kv, dtype, cols, B = sizes
    if T and B:
        rc, _ = _chunk(lib, T=T, heads=heads, kv=kv, dtype=dtype, cols=cols, B=B, q_ld=1 << 18, k_ld=1 << 18, v_ld=1 << 18)
        assert rc in (1, 4) and "null pointer" not in lib.uocr_last_error().decode()
    assert lib.uocr_paged_chunk_workspace_bytes(T, heads, kv, dtype, cols, B) == 0
    assert lib.uocr_paged_chunk_workspace_bytes(4, 4, 2, 0, 3, 2) > 0
