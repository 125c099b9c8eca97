"""Lengths that the page table does not cover, and rows that a call does not take."""

import numpy as np
import pytest

from bobcat_b200 import F16, I8, KvRows, errors
from kv_pool_cases import Pool, attention
from test_attention_paged_gpu import MARK, attend, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hint", [1, 1000])
@pytest.mark.parametrize("fmt", [F16, I8])
@pytest.mark.parametrize("kv, heads, hd", [(2, 4, 64), (1, 8, 128), (1, 3, 256)])
@pytest.mark.parametrize("news", [[1, 1], [50, 20], [3, 40]])
@pytest.mark.parametrize("length", [81, 95, 140])
def test_rows_behind_the_table_attend_to_what_it_holds(cuda, length, news, kv, heads, hd, fmt, hint):
    """A table of five pages of 16 and a longer sequence: each row sees the keys up to its own position that the table has, and the wait says so."""
    case = Pool(cuda, fmt, 16, kv, hd, [80, 40], np.random.default_rng(70), spare_columns=0)
    case.fill(np.random.default_rng(71))
    case.upload()
    assert case.max_pages == 5
    n = sum(news)
    q = (np.random.default_rng(72).standard_normal((n + 1, heads * hd)) * 1.5).astype(np.float32)
    qb, out = cuda.buffer_from(q), cuda.buffer_from(np.full(q.shape, MARK, dtype=np.float32))
    scratch = cuda.new_buffer(4 * cuda.attention_paged_scratch_floats(heads, kv, hd))
    rows = case.rows(news, n_rows=n + 1, lens=[length, 40], max_queries=hint)
    cuda.begin()
    cuda.attention_paged(case.pool, rows, qb, scratch, out, heads, heads * hd, hd)
    with pytest.raises(errors.OutOfBounds, match="positions"):
        cuda.end()
    got = cuda.read(out, np.zeros_like(q))
    for s, at, first, held in ((0, 0, length - news[0], 80), (1, news[0], 40 - news[1], 40)):
        rows_of = slice(at, at + news[s])
        want, bound = attention(q[rows_of].reshape(-1, heads, hd), case.context(case.k_raw, s, held), case.context(case.v_raw, s, held), first)
        assert (np.abs(got[rows_of].reshape(-1, heads, hd) - want) <= bound).all()
    assert (got[n:] == MARK).all()


@pytest.mark.parametrize("fmt", [F16, I8])
def test_rows_behind_the_table_are_not_written(cuda, fmt):
    case = Pool(cuda, fmt, 16, 2, 64, [80, 40], np.random.default_rng(73), spare_columns=0)
    x = np.random.default_rng(74).standard_normal((130, 256)).astype(np.float32)
    pool, rows, xb = case.upload(), case.rows([90, 40], lens=[90, 40]), cuda.buffer_from(x)
    cuda.begin()
    cuda.kv_write(pool, rows, xb, xb.floats(128), 256, 256)
    with pytest.raises(errors.OutOfBounds, match="positions"):
        cuda.end()
    for s, row0, n in ((0, 0, 80), (1, 90, 40)):
        for pos in range(n):
            case.put(case.k_raw, s, pos, x[row0 + pos, :128].reshape(2, 64))
            case.put(case.v_raw, s, pos, x[row0 + pos, 128:].reshape(2, 64))
    k_now, v_now = case.download()
    assert np.array_equal(k_now, case.k_raw) and np.array_equal(v_now, case.v_raw)


@pytest.mark.parametrize("hint", [1, 1000])
@pytest.mark.parametrize("fmt", [F16, I8])
@pytest.mark.parametrize("end", [41, 1 << 24, (1 << 31) + 5, (1 << 32) - 1])
def test_rows_of_a_sequence_that_a_call_does_not_take(cuda, end, fmt, hint):
    """A sequence of more rows than the call takes, and than positions: those that it takes lie before the first position, or at it."""
    case = Pool(cuda, fmt, 16, 2, 64, [40], np.random.default_rng(75))
    case.fill(np.random.default_rng(76))
    case.upload()
    q = np.random.default_rng(77).standard_normal((40, 4 * 64)).astype(np.float32)
    c = cuda
    rows = KvRows(1, 40, hint, case.max_pages, c.buffer_from(case.table), c.buffer_from(np.array([0, end], dtype=np.uint32)), c.buffer_from(np.array([40], dtype=np.uint32)))
    got = attend(cuda, case, [40], 4, q, rows=rows)
    if end == 41:  # row r is position r - 1
        assert (got[0] == 0).all()
        check(case, [39], 4, q[1:], got[1:], lens=[39])
    else:
        assert (got == 0).all()
    back = cuda.buffer_from(np.full((40, 128), 9.0, dtype=np.float32))
    cuda.begin()
    cuda.kv_read(case.pool, rows, back, None, False, 128, 128)
    cuda.end()
    want = np.zeros((40, 128), dtype=np.float32)
    if end == 41:
        want[1:] = np.stack([case.get(case.k_raw, 0, pos, np.float32).reshape(-1) for pos in range(39)])
    assert np.array_equal(cuda.read(back, np.zeros_like(want)), want)
