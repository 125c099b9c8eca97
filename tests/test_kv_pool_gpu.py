"""Rows into the pages of a key/value pool and back: bytes and scales equal the stored form worked out in 64 bits, whatever is no row's
stays as it was."""

import numpy as np
import pytest

from bobcat_b200 import F16, I8, KvPool, KvRows, errors
from kv_pool_cases import Pool, stored

pytestmark = pytest.mark.gpu


def write(cuda, case, news, n_rows, seed, rows_of=None, special=None, pad=0):
    """Writes rows of a [rows][before | keys | values | pad] product; the pool's bytes after it, and the rows."""
    rng = np.random.default_rng(seed)
    width = case.kv * case.hd
    x = rng.standard_normal((max(n_rows, 1), 8 + 2 * width + pad)).astype(np.float32)
    if special is not None:
        special(x[:, 8:])
    pool, rows, xb = case.upload(), case.rows(news, n_rows) if rows_of is None else rows_of, cuda.buffer_from(x)
    cuda.begin()
    cuda.kv_write(pool, rows, xb.floats(8), xb.floats(8 + width), x.shape[1], x.shape[1])
    cuda.end()
    starts = np.concatenate([[0], np.cumsum(news)])
    for s, n in enumerate(news):
        for i in range(n):
            pos = case.lens[s] - n + i
            if pos < 0 or starts[s] + i >= n_rows:
                continue
            row = x[starts[s] + i, 8:]
            case.put(case.k_raw, s, pos, row[:width].reshape(case.kv, case.hd))
            case.put(case.v_raw, s, pos, row[width:2 * width].reshape(case.kv, case.hd))
    return x, rows


@pytest.mark.parametrize("fmt", [F16, I8])
@pytest.mark.parametrize("page_size, kv, hd, lens, news, spare_rows", [
    (16, 8, 64, [301], [1], 0),
    (16, 2, 64, [5, 0, 40, 17], [5, 0, 3, 1], 4),       # a sequence without rows, rows behind the last sequence
    (32, 3, 128, [33, 64, 31], [33, 1, 31], 1),         # an odd number of heads
    (64, 4, 256, [70, 1, 200], [6, 1, 129], 0),
    (128, 1, 64, [256], [256], 0),
    (256, 2, 128, [300, 257], [300, 2], 0),
    (16, 40, 256, [9, 4], [9, 4], 3),                   # more heads than a CTA has threads for in a round
    (16, 2, 64, [2, 3], [5, 3], 0),                     # more rows than positions: the first three have no place
    (16, 1, 64, list(range(1, 201)), [1] * 200, 9),     # more sequences than a warp looks at at once
])
def test_rows_are_stored_and_read(cuda, fmt, page_size, kv, hd, lens, news, spare_rows):
    case = Pool(cuda, fmt, page_size, kv, hd, lens, np.random.default_rng(1))
    n_rows = sum(news) + spare_rows
    x, rows = write(cuda, case, news, n_rows, seed=kv + hd, pad=4)
    k_now, v_now = case.download()
    assert np.array_equal(k_now, case.k_raw) and np.array_equal(v_now, case.v_raw)

    width = kv * hd
    starts = np.concatenate([[0], np.cumsum(news)])
    for half, dtype in ((False, np.float32), (True, np.float16)):
        mark = dtype(-77)
        k_out, v_out = (cuda.buffer_from(np.full((n_rows, width + 8), mark, dtype=dtype)) for _ in range(2))
        cuda.begin()
        cuda.kv_read(case.pool, rows, k_out, v_out, half, width + 8, width + 8)
        cuda.end()
        for out, raw in ((k_out, case.k_raw), (v_out, case.v_raw)):
            want = np.full((n_rows, width + 8), mark, dtype=dtype)
            for s, n in enumerate(news):
                for i in range(n):
                    pos = lens[s] - n + i
                    want[starts[s] + i, :width] = 0 if pos < 0 else case.get(raw, s, pos, np.float32).reshape(-1).astype(dtype)
            assert np.array_equal(cuda.read(out, np.zeros_like(want)), want)


@pytest.mark.parametrize("fmt", [F16, I8])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_numbers_at_the_edges(cuda, fmt, hd):
    """Zeros, rows whose scale is no normal number, the largest floats, ties, infinities and NaN."""
    case = Pool(cuda, fmt, 16, 1, hd, [16], np.random.default_rng(2))

    def special(x):  # [16][keys | values]
        x[0] = 0.0
        x[1] = 1e-40
        x[2, :hd] = np.linspace(-1, 1, hd) * 1e-36      # a scale below the normal numbers
        x[3, :hd] = np.linspace(-1, 1, hd) * 1.6e-36    # and just above them
        x[4] = np.sign(x[4]) * np.float32(3.4e38)
        x[5, :hd] = 127.0 - np.arange(hd) / 2.0         # scale 1: whole numbers and halves between them
        x[6, :hd] = -127.0 + np.arange(hd) / 2.0
        x[7, :hd] = (np.arange(hd) - hd // 2) * np.float32(0.1)
        x[8, 3] = np.inf
        x[9, hd + 5] = np.nan
        x[10, 7] = -np.inf
        x[11, :hd] = np.float32(127) * np.float32(0.3) - np.arange(hd) * np.float32(0.15)
        x[12, :hd] = 70000.0                            # above the largest half
        x[13, :hd] = np.where(np.arange(hd) % 2, 1.0, -1.0) * np.float32(2.0) ** -25

    write(cuda, case, [16], 16, seed=3, special=special)
    k_now, v_now = case.download()
    if fmt == I8:
        assert np.array_equal(k_now, case.k_raw) and np.array_equal(v_now, case.v_raw)
        return
    for now, want in ((k_now, case.k_raw), (v_now, case.v_raw)):
        a, b = now.view(np.float16), want.view(np.float16)
        assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(a[~np.isnan(a)], b[~np.isnan(b)])


def test_quotients_beside_a_half(cuda):
    """Elements within a few last places of the middle between two whole numbers, on either side of it."""
    rng = np.random.default_rng(4)
    case = Pool(cuda, I8, 64, 8, 64, [512], np.random.default_rng(5))

    def special(x):
        for row in x:
            for head in row[:2 * 8 * 64].reshape(-1, 64):
                top = np.float32(rng.uniform(0.5, 2.0))
                scale = np.float32(np.float64(top) / 127.0)
                middle = ((rng.integers(-126, 126, 64) + 0.5) * np.float64(scale)).astype(np.float32)
                steps = rng.integers(-2, 3, 64)
                head[:] = (middle.view(np.int32) + steps.astype(np.int32)).view(np.float32)
                head[0] = top

    write(cuda, case, [512], 512, seed=6, special=special)
    k_now, v_now = case.download()
    assert np.array_equal(k_now, case.k_raw) and np.array_equal(v_now, case.v_raw)


def test_keys_or_values_alone(cuda):
    case = Pool(cuda, I8, 16, 2, 64, [20], np.random.default_rng(7))
    case.fill(np.random.default_rng(8))
    pool, rows = case.upload(), case.rows([20])
    out = cuda.new_buffer(20 * 128 * 4)
    for which, raw in ((0, case.k_raw), (1, case.v_raw)):
        cuda.begin()
        cuda.kv_read(pool, rows, out if which == 0 else None, out if which == 1 else None, False, 128, 128)
        cuda.end()
        want = np.stack([case.get(raw, 0, pos, np.float32).reshape(-1) for pos in range(20)])
        assert np.array_equal(cuda.read(out, np.zeros_like(want)), want)


def test_pages_that_are_not_there(cuda):
    """A page number outside the pool, and a sequence longer than its table: nothing is written or read there, the wait says so, once."""
    case = Pool(cuda, I8, 16, 2, 64, [40, 10], np.random.default_rng(9), spare_columns=0)
    case.table[0, 1] = case.n_pages  # positions 16 .. 31
    rng = np.random.default_rng(10)
    x = rng.standard_normal((50, 256)).astype(np.float32)
    pool, rows, xb = case.upload(), case.rows([40, 10]), cuda.buffer_from(x)
    cuda.begin()
    cuda.kv_write(pool, rows, xb, xb.floats(128), 256, 256)
    with pytest.raises(errors.OutOfBounds, match="page"):
        cuda.end()
    for r, (s, pos) in enumerate([(0, i) for i in range(40)] + [(1, i) for i in range(10)]):
        if s == 0 and 16 <= pos < 32:
            continue
        case.put(case.k_raw, s, pos, x[r, :128].reshape(2, 64))
        case.put(case.v_raw, s, pos, x[r, 128:].reshape(2, 64))
    k_now, v_now = case.download()
    assert np.array_equal(k_now, case.k_raw) and np.array_equal(v_now, case.v_raw)
    out = cuda.buffer_from(np.full((50, 128), 9.0, dtype=np.float32))
    cuda.begin()
    cuda.kv_read(pool, rows, out, None, False, 128, 128)
    with pytest.raises(errors.OutOfBounds, match="page"):
        cuda.end()
    got = cuda.read(out, np.zeros((50, 128), dtype=np.float32))
    assert (got[16:32] == 0).all() and (got[:16] != 0).any()

    long = case.rows([0, 2], lens=[0, 49])  # the table has three pages of 16
    out = cuda.buffer_from(np.full((2, 128), 9.0, dtype=np.float32))
    case.table[1, 1:] = 0
    long = case.rows([0, 2], lens=[0, 49])
    cuda.begin()
    cuda.kv_read(pool, long, out, None, False, 128, 128)
    with pytest.raises(errors.OutOfBounds, match="positions"):
        cuda.end()
    assert (cuda.read(out, np.zeros((2, 128), dtype=np.float32))[1] == 0).all()
    cuda.begin()
    cuda.end()  # reported once


def test_refusals(cuda):
    case = Pool(cuda, I8, 16, 2, 64, [20], np.random.default_rng(11))
    pool, rows = case.upload(), case.rows([20])
    x = cuda.new_buffer(20 * 128 * 4)
    with pytest.raises(errors.NotRecording):
        cuda.kv_write(pool, rows, x, x, 128, 128)
    cuda.begin()

    def refused(error, pool=pool, rows=rows, k=x, v=x, k_stride=128, v_stride=128):
        with pytest.raises(error):
            cuda.kv_write(pool, rows, k, v, k_stride, v_stride)
        with pytest.raises(error):
            cuda.kv_read(pool, rows, k, v, False, k_stride, v_stride)

    def pool_with(**changes):
        fields = dict(fmt=I8, n_pages=case.n_pages, page_size=16, n_kv_heads=2, head_dim=64, k=case.k, v=case.v)
        fields.update(changes)
        return KvPool(*fields.values())

    def rows_with(**changes):
        fields = dict(n_seqs=1, n_rows=20, max_queries=20, max_pages=case.max_pages, table=rows.holds[0], starts=rows.holds[1], lens=rows.holds[2])
        fields.update(changes)
        return KvRows(*fields.values())

    refused(errors.Unsupported, pool=pool_with(fmt=8))
    for changes in (dict(page_size=8), dict(page_size=24), dict(page_size=512), dict(n_kv_heads=0), dict(n_kv_heads=1025), dict(head_dim=96), dict(head_dim=512)):
        refused(errors.AttentionLimits, pool=pool_with(**changes))
    refused(errors.Argument, pool=pool_with(n_pages=0))
    refused(errors.OutOfBounds, pool=pool_with(n_pages=case.n_pages + 1))
    refused(errors.OutOfBounds, pool=pool_with(n_pages=0xFFFFFFFF))
    refused(errors.OutOfBounds, pool=pool_with(k=case.k.at(16)))
    refused(errors.Argument, pool=pool_with(n_pages=1, v=case.v.at(8)))
    refused(errors.Argument, pool=pool_with(k=None))
    for changes in (dict(n_seqs=0), dict(n_seqs=65536), dict(max_pages=0), dict(max_pages=(1 << 27) + 1), dict(max_queries=0), dict(n_rows=(1 << 24) + 1)):
        refused(errors.Argument, rows=rows_with(**changes))
    refused(errors.OutOfBounds, rows=rows_with(n_seqs=2))
    refused(errors.OutOfBounds, rows=rows_with(max_pages=case.max_pages + 1))
    refused(errors.OutOfBounds, rows=rows_with(starts=rows.holds[1].at(4)))
    refused(errors.Argument, rows=rows_with(max_pages=1, table=rows.holds[0].at(2)))
    refused(errors.Argument, rows=rows_with(lens=None))
    refused(errors.OutOfBounds, rows=rows_with(n_rows=21))
    refused(errors.Argument, k_stride=124)
    refused(errors.Argument, v_stride=130)
    refused(errors.Argument, k=x.at(4))
    refused(errors.OutOfBounds, v=x.at(16))
    refused(errors.OutOfBounds, k_stride=132)
    with pytest.raises(errors.Argument):
        cuda.kv_write(pool, rows, None, x, 128, 128)
    with pytest.raises(errors.Argument):
        cuda.kv_read(pool, rows, None, None, False, 128, 128)
    with pytest.raises(errors.Argument):
        cuda.kv_read(pool, rows_with(n_rows=1), x, x, True, 132, 128)  # halves: 8 to 16 bytes
    cuda.end()


def test_buffers_over_memory_of_the_caller(cuda):
    torch = pytest.importorskip("torch")
    t = torch.arange(1024, dtype=torch.float32, device="cuda")
    torch.cuda.synchronize()
    b = cuda.buffer_at(t.data_ptr(), t.numel() * 4)
    assert len(b) == 4096 and b.device_ptr == t.data_ptr()
    assert np.array_equal(cuda.read(b, np.zeros(1024, dtype=np.float32)), np.arange(1024, dtype=np.float32))
    cuda.write(b.floats(4), np.full(4, -1, dtype=np.float32))
    assert t[4:8].tolist() == [-1.0] * 4
    with pytest.raises(errors.OutOfBounds):
        cuda.read(b, np.zeros(1025, dtype=np.float32))
    b.free()
    assert t[:4].tolist() == [0.0, 1.0, 2.0, 3.0]  # still the caller's
    with pytest.raises(errors.Argument):
        cuda.buffer_at(t.data_ptr() + 16, 64)
    with pytest.raises(errors.Argument):
        cuda.buffer_at(0, 64)
    host = torch.zeros(64).pin_memory()
    with pytest.raises(errors.Argument):
        cuda.buffer_at(host.data_ptr() // 256 * 256, 64)


@pytest.mark.parametrize("n_seqs", [255, 256, 257, 300, 1023, 1056, 5000])
def test_rows_find_their_sequence_among_many(cuda, n_seqs):
    rng = np.random.default_rng(n_seqs)
    news = [int(n) for n in rng.choice([0, 0, 1, 1, 2, 5], size=n_seqs)]
    lens = [n + int(rng.integers(0, 20)) for n in news]
    case = Pool(cuda, F16, 16, 1, 64, lens, rng)
    pool, n = case.upload(), sum(news)
    x = rng.standard_normal((n + 3, 64)).astype(np.float16).astype(np.float32)
    starts = np.concatenate([[0], np.cumsum(news)])
    rows, xb = case.rows(news, n_rows=n + 3), cuda.buffer_from(x)
    back = cuda.buffer_from(np.full((n + 3, 64), 9.0, dtype=np.float32))
    cuda.begin()
    cuda.kv_write(pool, rows, xb, xb, 64, 64)
    cuda.kv_read(pool, rows, back, None, False, 64, 64)
    cuda.end()
    for s, m in enumerate(news):
        for i in range(m):
            case.put(case.k_raw, s, lens[s] - m + i, x[starts[s] + i].reshape(1, 64))
    assert np.array_equal(case.download()[0], case.k_raw)
    got = cuda.read(back, np.zeros_like(x))
    assert np.array_equal(got[:n], x[:n]) and (got[n:] == 9.0).all()


def test_stored_is_what_the_formula_says():
    """The numpy form that the tests compare with: halfway cases to even, exact zeros."""
    held, scales = stored(np.array([[127.0, 0.5, 1.5, -2.5]], dtype=np.float32), I8)
    assert scales.tolist() == [1.0] and (held.astype(int) - 128).tolist() == [[127, 0, 2, -2]]
