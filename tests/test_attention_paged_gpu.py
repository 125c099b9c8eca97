"""Attention of the new rows of several sequences over a pool of key/value pages, against 64 bits, within a bound worked out from the
operands (kv_pool_cases.attention). Every position that is not a sequence's holds NaN, in the pages' elements and scales alike."""

import numpy as np
import pytest

from bobcat_b200 import Cuda, F16, I8, KvPool, KvRows, errors
from kv_pool_cases import Pool, attention

pytestmark = pytest.mark.gpu

MARK = np.float32(-55.0)


def build(cuda, fmt, page_size, kv, hd, lens, seed, amplitude=1.0):
    case = Pool(cuda, fmt, page_size, kv, hd, lens, np.random.default_rng(seed))
    case.fill(np.random.default_rng(seed + 1), amplitude)
    return case


def attend(cuda, case, news, heads, q, rows=None, q_head_stride=None, offset=0):
    """q [rows][stride]; rows of no sequence keep MARK."""
    hd, n_rows = case.hd, q.shape[0]
    rows = case.rows(news, n_rows) if rows is None else rows
    qb, out = cuda.buffer_from(q), cuda.buffer_from(np.full((n_rows, heads * hd), MARK, dtype=np.float32))
    scratch = cuda.buffer_from(np.full(cuda.attention_paged_scratch_floats(heads, case.kv, hd), np.nan, dtype=np.float32))
    cuda.begin()
    cuda.attention_paged(case.pool, rows, qb.floats(offset), scratch, out, heads, q.shape[1], q_head_stride or hd)
    cuda.end()
    return cuda.read(out, np.zeros((n_rows, heads * hd), dtype=np.float32))


def check(case, news, heads, q, got, q_head_stride=None, offset=0, lens=None):
    hd, at = case.hd, 0
    stride = q_head_stride or hd
    for s, n in enumerate(news):
        length = (lens or case.lens)[s]
        k, v = case.context(case.k_raw, s, length), case.context(case.v_raw, s, length)
        rows = np.stack([q[at:at + n, offset + h * stride:offset + h * stride + hd] for h in range(heads)], axis=1) if n else np.zeros((0, heads, hd))
        want, bound = attention(rows, k, v, length - n)
        have = got[at:at + n].reshape(n, heads, hd)
        assert np.isfinite(have).all(), s
        assert (np.abs(have - want) <= bound).all(), (s, n, length, (np.abs(have - want) / np.maximum(bound, 1e-30)).max())
        at += n
    assert (got[at:] == MARK).all()


TOKENS = [
    (16, 2, 2, 64, [1]),
    (16, 4, 2, 64, [15, 16, 17, 1, 127, 128, 129]),
    (32, 8, 8, 64, [301, 0, 33]),                 # a sequence without positions
    (64, 16, 2, 128, [257, 64, 5]),
    (16, 3, 3, 128, [100, 700]),
    (128, 8, 1, 256, [1, 600]),
    (256, 14, 2, 256, [513, 255]),
    (64, 32, 8, 64, [5000]),                      # over many CTAs
    (16, 12, 4, 64, list(range(1, 70))),
]


@pytest.mark.parametrize("fmt", [F16, I8])
@pytest.mark.parametrize("page_size, heads, kv, hd, lens", TOKENS)
def test_single_tokens(cuda, fmt, page_size, heads, kv, hd, lens):
    case = build(cuda, fmt, page_size, kv, hd, lens, seed=heads + hd)
    case.upload()
    news = [1] * len(lens)
    q = (np.random.default_rng(hd).standard_normal((len(lens) + 2, heads * hd)) * 1.5).astype(np.float32)  # two rows behind the last sequence
    check(case, news, heads, q, attend(cuda, case, news, heads, q))


CHUNKS = [
    (16, 4, 2, 64, [(2, 2), (3, 90)]),
    (16, 2, 2, 64, [(5, 3), (4, 4)]),             # rows before the first position see nothing
    (32, 8, 2, 64, [(40, 40), (0, 50), (1, 200), (65, 130)]),
    (64, 8, 8, 64, [(129, 129), (7, 400)]),
    (64, 8, 1, 128, [(17, 17), (16, 300), (1, 1)]),
    (16, 4, 4, 128, [(130, 260)]),
    (128, 6, 2, 256, [(33, 33), (2, 300), (50, 190)]),
    (256, 4, 1, 256, [(64, 513)]),
    (32, 10, 2, 128, [(13, 70), (1, 129), (100, 227), (31, 31)]),
]


@pytest.mark.parametrize("fmt", [F16, I8])
@pytest.mark.parametrize("page_size, heads, kv, hd, seqs", CHUNKS)
def test_chunks(cuda, fmt, page_size, heads, kv, hd, seqs):
    news, lens = [n for n, _ in seqs], [length for _, length in seqs]
    case = build(cuda, fmt, page_size, kv, hd, lens, seed=heads + hd + 7)
    case.upload()
    q = (np.random.default_rng(hd + 1).standard_normal((sum(news) + 3, heads * hd)) * 1.5).astype(np.float32)
    check(case, news, heads, q, attend(cuda, case, news, heads, q))


@pytest.mark.parametrize("fmt", [F16, I8])
@pytest.mark.parametrize("page_size, heads, kv, hd, seqs", [
    (64, 8, 8, 64, [(70, 30000)]),                # one head a group: two row tiles of 235 key tiles and eight heads over the device
    (128, 16, 8, 128, [(40, 40000)]),
    (256, 8, 4, 256, [(20, 20000)]),              # key tiles of 64
    (16, 16, 4, 128, [(3, 9000), (90, 17000), (1, 12000), (5, 33)]),
])
def test_long_contexts(cuda, fmt, page_size, heads, kv, hd, seqs):
    """Many key tiles to a CTA, so that every ring of the pipeline wraps many times."""
    news, lens = [n for n, _ in seqs], [length for _, length in seqs]
    case = Pool(cuda, fmt, page_size, kv, hd, lens, np.random.default_rng(30))
    case.fill_at_once(np.random.default_rng(31))
    case.upload()
    q = (np.random.default_rng(32).standard_normal((sum(news), heads * hd)) * 1.5).astype(np.float32)
    check(case, news, heads, q, attend(cuda, case, news, heads, q))


@pytest.mark.parametrize("fmt", [F16, I8])
@pytest.mark.parametrize("news", [[1, 1], [70, 9]])
def test_what_the_caller_says_of_the_rows_is_no_more_than_a_hint(cuda, fmt, news):
    case = build(cuda, fmt, 32, 2, 128, [150, 37], seed=3)
    case.upload()
    q = np.random.default_rng(5).standard_normal((sum(news), 8 * 128)).astype(np.float32)
    for hint in (1, 2, 1000):
        check(case, news, 8, q, attend(cuda, case, news, 8, q, rows=case.rows(news, max_queries=hint)))


@pytest.mark.parametrize("fmt", [F16, I8])
@pytest.mark.parametrize("news", [[1, 1], [40, 3]])
def test_strided_queries(cuda, fmt, news):
    """Queries and gates of a head side by side, rows in the middle of a wider product."""
    case = build(cuda, fmt, 16, 2, 64, [90, 33], seed=6)
    case.upload()
    q = np.random.default_rng(7).standard_normal((sum(news), 8 + 4 * 128 + 12)).astype(np.float32)
    got = attend(cuda, case, news, 4, q, q_head_stride=128, offset=8, rows=case.rows(news))
    check(case, news, 4, q, got, q_head_stride=128, offset=8)


@pytest.mark.parametrize("fmt", [F16, I8])
@pytest.mark.parametrize("news", [[1], [70]])
@pytest.mark.parametrize("k_size, v_size, q_size", [(1e-4, 1e-4, 1e4), (100.0, 1e-4, 1e-3), (0.02, 100.0, 30.0), (1e-3, 1.0, 1e-6)])
def test_magnitudes(cuda, fmt, news, k_size, v_size, q_size):
    """Scores and values keep their bits however large or small the operands are. (Halves of cache elements below 2^-14 are what they are: the
    expectation takes the stored values.)"""
    case = Pool(cuda, fmt, 64, 2, 128, [300], np.random.default_rng(8))
    rng = np.random.default_rng(9)
    for pos in range(300):
        size = 10.0 ** rng.uniform(-3, 0)  # positions differ among themselves too
        case.put(case.k_raw, 0, pos, (rng.standard_normal((2, 128)) * k_size).astype(np.float32))
        case.put(case.v_raw, 0, pos, (rng.standard_normal((2, 128)) * v_size * size).astype(np.float32))
    case.upload()
    q = (rng.standard_normal((news[0], 4 * 128)) * q_size).astype(np.float32)
    check(case, news, 4, q, attend(cuda, case, news, 4, q))


@pytest.mark.parametrize("fmt", [F16, I8])
def test_one_position_outweighs_the_rest(cuda, fmt):
    """Scores hundreds apart: the maximum moves late, and what came before weighs nothing."""
    case = Pool(cuda, fmt, 16, 1, 64, [400], np.random.default_rng(10))
    rng = np.random.default_rng(11)
    for pos in range(400):
        case.put(case.k_raw, 0, pos, np.full((1, 64), 0.05 * pos, dtype=np.float32))
        case.put(case.v_raw, 0, pos, (rng.standard_normal((1, 64)) * (1000.0 if pos < 200 else 1.0)).astype(np.float32))
    case.upload()
    for news in ([1], [130]):
        for sign in (1.0, -1.0):
            q = np.full((news[0], 2 * 64), sign * 4.0, dtype=np.float32)
            check(case, news, 2, q, attend(cuda, case, news, 2, q))


@pytest.mark.parametrize("fmt", [F16, I8])
def test_infinities_and_nan_of_later_positions_stay_where_they_are(cuda, fmt):
    """Rows before a position whose values or keys are not finite are not touched by it; rows from there on show it."""
    case = build(cuda, fmt, 16, 2, 64, [100], seed=12)
    bad = np.ones((2, 64), dtype=np.float32)
    bad[0, 5], bad[1, 9] = np.inf, np.nan
    case.put(case.v_raw, 0, 60, bad)
    case.put(case.k_raw, 0, 80, bad)
    case.upload()
    q = np.random.default_rng(13).standard_normal((90, 4 * 64)).astype(np.float32)
    got = attend(cuda, case, [90], 4, q)  # positions 10 .. 99
    k, v = case.context(case.k_raw, 0, 60), case.context(case.v_raw, 0, 60)
    want, bound = attention(q[:50].reshape(50, 4, 64), k, v, 10)
    assert (np.abs(got[:50].reshape(50, 4, 64) - want) <= bound).all()
    later = got[50:].reshape(40, 2, 2, 64)
    if fmt == F16:
        assert not np.isfinite(later[:, 0, :, 5]).any() and not np.isfinite(later[:, 1, :, 9]).any()
        clean = later[:20].copy()
        clean[:, 0, :, 5] = clean[:, 1, :, 9] = 0
        assert np.isfinite(clean).all()  # the other elements of those rows
    else:
        assert np.isnan(later).all()  # an 8-bit row with one such element reads as NaN
    assert not np.isfinite(got[70:].reshape(20, 2, 2, 64)[:, 1]).any()


@pytest.mark.parametrize("fmt", [F16, I8])
@pytest.mark.parametrize("news", [[1, 1], [50, 20]])
def test_a_page_that_is_not_there_is_left_out(cuda, fmt, news):
    case = build(cuda, fmt, 16, 1, 64, [70, 40], seed=14)
    hole = case.table.copy()
    hole[0, 1] = case.n_pages + 5
    case.upload()
    q = np.random.default_rng(15).standard_normal((sum(news), 2 * 64)).astype(np.float32)
    case.table, whole = hole, case.table
    rows = case.rows(news)
    case.table = whole
    qb, out = cuda.buffer_from(q), cuda.new_buffer(q.nbytes)
    scratch = cuda.new_buffer(4 * cuda.attention_paged_scratch_floats(2, 1, 64))
    cuda.begin()
    cuda.attention_paged(case.pool, rows, qb, scratch, out, 2, 128, 64)
    with pytest.raises(errors.OutOfBounds, match="page"):
        cuda.end()
    got = cuda.read(out, np.zeros_like(q))
    k, v = (np.delete(case.context(raw, 0, 70), np.arange(16, 32), axis=0) for raw in (case.k_raw, case.v_raw))
    for i in range(news[0]):
        pos = 70 - news[0] + i
        see = pos + 1 - max(0, min(pos + 1, 32) - 16)
        if see <= 0:
            continue
        want, bound = attention(q[i].reshape(1, 2, 64), k[:see], v[:see], see - 1)
        assert (np.abs(got[i].reshape(1, 2, 64) - want) <= bound).all(), i
    want, bound = attention(q[news[0]:].reshape(-1, 2, 64), case.context(case.k_raw, 1, 40), case.context(case.v_raw, 1, 40), 40 - news[1])
    assert (np.abs(got[news[0]:].reshape(-1, 2, 64) - want) <= bound).all()


@pytest.mark.parametrize("fmt", [F16, I8])
def test_pages_far_into_a_large_pool(cuda, fmt):
    """Byte offsets that do not fit 32 bits."""
    kv, hd, page_size, length, heads = 8, 256, 256, 600, 8
    page_bytes = cuda.kv_pool_bytes(fmt, 1, page_size, kv, hd)
    n_pages = (5 << 30) // page_bytes
    small = build(cuda, fmt, page_size, kv, hd, [length], seed=16)
    far = [n_pages - 2, n_pages - 1, (1 << 32) // page_bytes]
    k, v = cuda.new_buffer(n_pages * page_bytes), cuda.new_buffer(n_pages * page_bytes)
    for i, page in enumerate(far):
        cuda.write(k.at(page * page_bytes), small.k_raw[small.table[0, i]])
        cuda.write(v.at(page * page_bytes), small.v_raw[small.table[0, i]])
    pool = KvPool(fmt, n_pages, page_size, kv, hd, k, v)
    table = cuda.buffer_from(np.array([far], dtype=np.uint32))
    for n in (1, 40):
        rows = KvRows(1, n, n, 3, table, cuda.buffer_from(np.array([0, n], dtype=np.uint32)), cuda.buffer_from(np.array([length], dtype=np.uint32)))
        q = np.random.default_rng(17).standard_normal((n, heads * hd)).astype(np.float32)
        qb, out = cuda.buffer_from(q), cuda.new_buffer(q.nbytes)
        scratch = cuda.new_buffer(4 * cuda.attention_paged_scratch_floats(heads, kv, hd))
        back_k, back_v = cuda.new_buffer(n * kv * hd * 4), cuda.new_buffer(n * kv * hd * 4)
        cuda.begin()
        cuda.attention_paged(pool, rows, qb, scratch, out, heads, heads * hd, hd)
        cuda.kv_read(pool, rows, back_k, back_v, False, kv * hd, kv * hd)
        cuda.kv_write(pool, rows, back_k, back_v, kv * hd, kv * hd)  # to where they came from
        cuda.end()
        check(small, [n], heads, q, cuda.read(out, np.zeros_like(q)))
        want = np.stack([small.get(small.k_raw, 0, pos, np.float32).reshape(-1) for pos in range(length - n, length)])
        assert np.array_equal(cuda.read(back_k, np.zeros_like(want)), want)
    for buffer in (k, v):
        buffer.free()


@pytest.mark.parametrize("fmt", [F16, I8])
def test_a_conversation(cuda, fmt):
    """Prompts, then tokens, then a chunk beside tokens, of three sequences over one pool, two of them on shared pages: rows written, attended to
    in the same recording, and compared with what the whole contexts say; halves also with the attention over a cache of its own."""
    kv, hd, heads, page_size = 2, 64, 8, 16
    rng = np.random.default_rng(18)
    case = Pool(cuda, fmt, page_size, kv, hd, [200, 200, 200], rng)
    case.table[2, :2] = case.table[1, :2]  # sequences 1 and 2 begin with the same 32 positions
    case.upload()
    width, lens = kv * hd, [0, 0, 0]
    scratch = cuda.new_buffer(4 * cuda.attention_paged_scratch_floats(heads, kv, hd))
    shared = None
    flat = [(cuda.new_buffer(256 * width * 2), cuda.new_buffer(256 * width * 2)) for _ in range(3)]
    for news in ([70, 32, 0], [0, 0, 32], [1, 1, 1], [1, 0, 1], [1, 45, 1], [4, 4, 3], [60, 1, 1]):
        n = sum(news)
        qkv = rng.standard_normal((n, heads * hd + 2 * width)).astype(np.float32)
        if news[1] == 32:
            shared = qkv[70:102, heads * hd:].copy()
        if news == [0, 0, 32]:
            qkv[:, heads * hd:] = shared  # written again, the same
        lens = [a + b for a, b in zip(lens, news)]
        rows = case.rows(news, lens=lens)
        xb, out = cuda.buffer_from(qkv), cuda.new_buffer(n * heads * hd * 4)
        cuda.begin()
        cuda.kv_write(case.pool, rows, xb.floats(heads * hd), xb.floats(heads * hd + width), qkv.shape[1], qkv.shape[1])
        cuda.attention_paged(case.pool, rows, xb, scratch, out, heads, qkv.shape[1], hd)
        cuda.end()
        at = 0
        for s, m in enumerate(news):
            for i in range(m):
                case.put(case.k_raw, s, lens[s] - m + i, qkv[at + i, heads * hd:heads * hd + width].reshape(kv, hd))
                case.put(case.v_raw, s, lens[s] - m + i, qkv[at + i, heads * hd + width:].reshape(kv, hd))
            at += m
        got = cuda.read(out, np.zeros((n, heads * hd), dtype=np.float32))
        check(case, news, heads, qkv, got, lens=lens)
        if fmt == F16:
            at = 0
            for s, m in enumerate(news):
                if m == 0:
                    continue
                for which, first in zip(flat[s], (heads * hd, heads * hd + width)):
                    cuda.write(which.at((lens[s] - m) * width * 2), qkv[at:at + m, first:first + width].astype(np.float16))
                need = cuda.new_buffer(4 * cuda.attention_scratch_floats(heads, hd, 256, m))
                qb, one = cuda.buffer_from(qkv[at:at + m, :heads * hd]), cuda.new_buffer(m * heads * hd * 4)
                cuda.begin()
                cuda.attention(qb, flat[s][0], flat[s][1], True, need, one, heads, kv, hd, lens[s] - m, m, 256)
                cuda.end()
                assert np.abs(cuda.read(one, np.zeros((m, heads * hd), dtype=np.float32)) - got[at:at + m]).max() < 1e-5
                at += m


@pytest.mark.parametrize("fmt", [F16, I8])
@pytest.mark.parametrize("hint", [64, 4])
def test_captured_calls_follow_the_lengths(fmt, hint):
    """A step captured once and replayed after the lengths, the tables and the rows have changed on the device; a second graph beside it with a
    scratch of its own, on another stream."""
    torch = pytest.importorskip("torch")
    kv, hd, heads = 2, 128, 8
    graphs = []
    for which in range(2):
        stream = torch.cuda.Stream()
        cuda = Cuda.open(0, stream.cuda_stream)
        case = build(cuda, fmt, 32, kv, hd, [300, 150, 40], seed=20 + which)
        case.upload()
        q = torch.zeros(64, heads * hd, device="cuda")
        out = torch.full((64, heads * hd), float(MARK), device="cuda")
        words = {n: torch.from_numpy(a.view(np.int32).copy()).cuda() for n, a in
                 dict(table=case.table, starts=np.array([0, 1, 2, 3], dtype=np.uint32), lens=np.array([300, 150, 40], dtype=np.uint32)).items()}
        torch.cuda.synchronize()
        at = {n: cuda.buffer_at(t.data_ptr(), t.numel() * 4) for n, t in dict(words, q=q, out=out).items()}
        rows = KvRows(3, 64, hint, case.max_pages, at["table"], at["starts"], at["lens"])
        scratch = cuda.new_buffer(4 * cuda.attention_paged_scratch_floats(heads, kv, hd))
        call = lambda: cuda.attention_paged(case.pool, rows, at["q"], scratch, at["out"], heads, heads * hd, hd)  # noqa: E731
        cuda.begin()
        call()
        cuda.end()
        cuda.begin()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
        cuda.end()
        graphs.append((stream, cuda, case, graph, q, out, words, at, scratch))
    rng = np.random.default_rng(21)
    for news, lens in (([1, 1, 1], [300, 150, 40]), ([60, 1, 0], [290, 12, 0]), ([1, 3, 33], [1, 140, 33])):
        staged = []
        for stream, cuda, case, graph, q, out, words, _, _ in graphs:
            x = (rng.standard_normal((64, heads * hd)) * 1.5).astype(np.float32)
            staged.append(x)
            q.copy_(torch.from_numpy(x))
            out.fill_(float(MARK))
            words["starts"].copy_(torch.tensor([0] + list(np.cumsum(news)), dtype=torch.int32))
            words["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize()
        for stream, cuda, case, graph, *_ in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for x, (stream, cuda, case, graph, q, out, *_) in zip(staged, graphs):
            check(case, news, heads, x, out.cpu().numpy(), lens=lens)
    for stream, cuda, *_ in graphs:
        cuda.close()


def test_attention_refusals(cuda):
    case = build(cuda, F16, 16, 2, 64, [20], seed=22)
    pool, rows, no_rows = case.upload(), case.rows([1]), case.rows([0], 0)
    need = cuda.attention_paged_scratch_floats(8, 2, 64)
    q, out, scratch = cuda.new_buffer(8 * 64 * 4), cuda.new_buffer(8 * 64 * 4), cuda.new_buffer(4 * need)
    with pytest.raises(errors.NotRecording):
        cuda.attention_paged(pool, rows, q, scratch, out, 8, 512, 64)
    cuda.begin()

    def refused(error, pool=pool, rows=rows, q=q, scratch=scratch, out=out, heads=8, q_stride=512, q_head_stride=64):
        with pytest.raises(error):
            cuda.attention_paged(pool, rows, q, scratch, out, heads, q_stride, q_head_stride)

    for heads in (0, 3, 18, 4 << 30 >> 1):
        refused(errors.AttentionLimits, heads=heads)
    refused(errors.Argument, q_stride=508)
    refused(errors.Argument, q_head_stride=60)
    refused(errors.Argument, q_head_stride=66)
    refused(errors.Argument, q_stride=514)
    refused(errors.Argument, q=q.at(8))
    refused(errors.Argument, out=None)
    refused(errors.Argument, scratch=scratch.at(8))
    refused(errors.OutOfBounds, scratch=scratch.at(16))
    refused(errors.OutOfBounds, out=out.at(16))
    refused(errors.OutOfBounds, q_head_stride=128, q_stride=1024)
    refused(errors.AttentionLimits, pool=KvPool(F16, case.n_pages, 16, 2, 32, case.k, case.v))
    other = Cuda.open(0)
    try:
        refused(errors.ForeignBuffer, out=other.new_buffer(4096))
    finally:
        other.close()
    cuda.attention_paged(pool, no_rows, q, scratch, out, 8, 512, 64)  # no rows: nothing to do
    cuda.end()


@pytest.mark.parametrize("fmt", [F16, I8])
@pytest.mark.parametrize("page_size, heads, kv, hd, seqs", [
    (16, 4, 2, 64, [(1, 1), (2, 40), (5, 3)]),
    (32, 8, 1, 64, [(3, 129)]),
    (64, 6, 2, 128, [(4, 300), (1, 65), (0, 20), (8, 9)]),
    (256, 8, 4, 128, [(2, 700)]),
    (128, 7, 1, 256, [(2, 64), (3, 65), (1, 500)]),
    (16, 5, 5, 256, [(9, 100), (1, 0)]),
])
def test_few_rows_either_way(cuda, fmt, page_size, heads, kv, hd, seqs):
    """The caller's word on the rows chooses the kernel: both say the same, within the bound."""
    news, lens = [n for n, _ in seqs], [length for _, length in seqs]
    case = build(cuda, fmt, page_size, kv, hd, lens, seed=heads + hd + 40)
    case.upload()
    q = (np.random.default_rng(hd + 41).standard_normal((sum(news) + 2, heads * hd)) * 1.5).astype(np.float32)
    for hint in (max(news), 32, 1000):
        check(case, news, heads, q, attend(cuda, case, news, heads, q, rows=case.rows(news, n_rows=q.shape[0], max_queries=hint)))


@pytest.mark.parametrize("fmt", [F16, I8])
@pytest.mark.parametrize("kv, heads, hd, n_seqs, hint", [(1, 2, 64, 97, 1000), (2, 8, 64, 330, 1000), (1, 1, 128, 64, 1000), (1, 2, 64, 700, 3), (4, 8, 256, 40, 1000)])
def test_many_sequences(cuda, fmt, kv, heads, hd, n_seqs, hint):
    """More sequences than lanes that look for a run's beginning; many of them without rows, rows of most too few to fill a row tile."""
    rng = np.random.default_rng(n_seqs)
    news = [int(n) for n in rng.choice([0, 1, 1, 2, 3, 7, 40], size=n_seqs)]
    news[0], news[-1], news[n_seqs // 2] = 0, 3, 150 if hint > 3 else 2
    lens = [n + int(rng.integers(0, 60)) if n else 5 for n in news]
    lens[1] = 900
    case = Pool(cuda, fmt, 16, kv, hd, lens, rng)
    case.fill_at_once(rng)
    case.upload()
    q = (rng.standard_normal((sum(news) + 1, heads * hd)) * 1.5).astype(np.float32)
    check(case, news, heads, q, attend(cuda, case, news, heads, q, rows=case.rows(news, n_rows=q.shape[0], max_queries=hint)))


@pytest.mark.parametrize("fmt", [F16, I8])
@pytest.mark.parametrize("kv, hd", [(8, 64), (4, 256)])
def test_row_tiles_cut_or_whole(cuda, fmt, kv, hd):
    """Short prompts, whose row tiles stay whole, and one beside them that makes equal runs the better choice."""
    rng = np.random.default_rng(hd)
    for news, lens in (([300], [300]), ([300, 1, 90], [300, 4000, 2500])):
        case = Pool(cuda, fmt, 32, kv, hd, lens, rng)
        case.fill_at_once(rng)
        case.upload()
        q = (rng.standard_normal((sum(news), 2 * kv * hd)) * 1.5).astype(np.float32)
        check(case, news, 2 * kv, q, attend(cuda, case, news, 2 * kv, q))
