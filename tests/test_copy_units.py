"""How an array of pages is copied, without a GPU: the rows that lie behind one another are one, and every piece that a thread takes starts on a multiple
of its size, whatever rows, strides and base the C ABI allows."""
import ctypes
import random

import pytest

from fused_attention_b200 import _lib


def described(**kw):
    area, out = _lib.CopyArea(**kw), (ctypes.c_uint32 * 4)()
    rc = _lib.load().fa_b200_describe_copy(ctypes.byref(area), out)
    return rc, list(out)


def rows_of(base, page, page_stride, n0, stride0, n1, stride1):
    return [base + page * page_stride + i * stride0 + j * stride1 for i in range(n0) for j in range(n1)]


def check(base, page_stride, stride0, stride1, n0, n1, row_bytes):
    """What is copied of three pages is what the area says; no piece lies across a boundary of its size."""
    rc, (m0, m1, row, unit) = described(base=base, page_stride=page_stride, stride0=stride0, stride1=stride1, n0=n0, n1=n1, row_bytes=row_bytes)
    assert rc == _lib.OK and unit in (4, 16) and row % unit == 0 and m0 * m1 * row == n0 * n1 * row_bytes
    for page in range(3):
        first = rows_of(base, page, page_stride, m0, stride0, m1, stride1)
        assert all(a % unit == 0 for a in first)
        want = {a + x for a in rows_of(base, page, page_stride, n0, stride0, n1, stride1) for x in range(0, row_bytes, 4)}
        assert {a + x for a in first for x in range(0, row, 4)} == want
    return unit


def test_rows_that_make_sixteen_bytes_together():
    """Short rows behind one another, on a base or with pages that are not multiples of 16 bytes."""
    assert check(base=0x1004, page_stride=64, stride0=0, stride1=8, n0=1, n1=2, row_bytes=8) == 4
    assert check(base=0x1000, page_stride=36, stride0=0, stride1=4, n0=1, n1=8, row_bytes=4) == 4
    assert check(base=0x1000, page_stride=48, stride0=24, stride1=8, n0=2, n1=2, row_bytes=8) == 4      # one row of 16 in every 24 bytes
    assert check(base=0x1000, page_stride=64, stride0=16, stride1=8, n0=2, n1=2, row_bytes=8) == 16     # and here all 32 in one
    assert check(base=0x1000, page_stride=1024, stride0=512, stride1=128, n0=2, n1=4, row_bytes=128) == 16


def test_any_area_that_is_taken():
    rng = random.Random(1)
    units = []
    for _ in range(3000):
        row, n0, n1 = 4 * rng.randint(1, 12), rng.randint(1, 4), rng.randint(1, 4)
        grain = 16 if row % 16 == 0 else 4
        stride1 = row + grain * rng.choice((0, 0, 1, 3))
        stride0 = n1 * stride1 + grain * rng.choice((0, 0, 1))
        page = n0 * stride0 + grain * rng.choice((0, 0, 1, 5))
        units.append(check(base=0x1000 + grain * rng.choice((0, 0, 1, 2, 3)), page_stride=page, stride0=stride0, stride1=stride1, n0=n0, n1=n1, row_bytes=row))
    assert units.count(4) > 300 and units.count(16) > 300


def test_refused():
    good = dict(base=0x1000, page_stride=64, stride0=32, stride1=16, n0=2, n1=2, row_bytes=16)
    assert described(**good) == (_lib.OK, [1, 1, 64, 16])
    for bad, rc in ((dict(base=None), _lib.ERR_NULL_POINTER), (dict(base=0x1008), _lib.ERR_ALIGNMENT), (dict(page_stride=72), _lib.ERR_ALIGNMENT),
                    (dict(stride1=8), _lib.ERR_ALIGNMENT), (dict(row_bytes=6), _lib.ERR_ALIGNMENT), (dict(row_bytes=8, base=0x1002), _lib.ERR_ALIGNMENT),
                    (dict(n0=0), _lib.ERR_SHAPE), (dict(row_bytes=0), _lib.ERR_SHAPE)):
        assert described(**{**good, **bad})[0] == rc
    assert _lib.load().fa_b200_describe_copy(None, (ctypes.c_uint32 * 4)()) == _lib.ERR_NULL_POINTER


@pytest.mark.gpu
def test_copied_on_the_gpu():
    """The areas above and random ones, several in a call, through the C entry."""
    import torch
    rng = random.Random(2)
    shapes = [(4, 64, 0, 8, 1, 2, 8), (0, 36, 0, 4, 1, 8, 4), (0, 48, 24, 8, 2, 2, 8), (0, 64, 16, 8, 2, 2, 8), (12, 36000, 9000, 4500, 2, 2, 4500), (8, 40, 0, 20, 1, 2, 20)]
    n, sources, targets = 9, [1, 8, 3], [0, 2, 7]
    for count in (1, len(shapes), 40):
        picked = [shapes[i % len(shapes)] for i in range(count)]
        held = [torch.randint(0, 256, (o + n * page + 16,), dtype=torch.uint8, device="cuda") for o, page, *_ in picked]
        before = [t.clone() for t in held]
        areas = (_lib.CopyArea * count)(*(_lib.CopyArea(t.data_ptr() + o, *rest) for t, (o, *rest) in zip(held, picked)))
        s, t = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (sources, targets))
        status = torch.zeros(2, dtype=torch.int32, device="cuda")
        rc = _lib.load().fa_b200_cache_copy(areas, count, n, s.data_ptr(), t.data_ptr(), len(sources), status.data_ptr(), 0, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert rc == _lib.OK and status.tolist() == [0, 0]
        for now, was, (o, page, stride0, stride1, n0, n1, row) in zip(held, before, picked):
            want = was.clone()
            for a, b in zip(sources, targets):
                for x, y in zip(rows_of(o, a, page, n0, stride0, n1, stride1), rows_of(o, b, page, n0, stride0, n1, stride1)):
                    want[y:y + row] = was[x:x + row]
            assert torch.equal(now, want)
