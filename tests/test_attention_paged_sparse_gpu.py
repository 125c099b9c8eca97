"""Calls of tens of thousands of sequences of which few have rows, or few have more than one: the walk from one to the next."""

import numpy as np
import pytest

from bobcat_b200 import F16, I8
from kv_pool_cases import Pool
from test_attention_paged_gpu import attend, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", [F16, I8])
@pytest.mark.parametrize("hint", [1, 1000])
@pytest.mark.parametrize("news", [{0: 300, 65534: 300}, {5: 1, 40000: 2, 65533: 1}, {31: 40, 32: 1, 33: 200, 30000: 3, 64000: 129}, {65534: 77}, {0: 500}])
def test_few_sequences_with_rows_among_many_without(cuda, news, hint, fmt):
    n_seqs = 65535
    rng = np.random.default_rng(90)
    all_news = [news.get(s, 0) for s in range(n_seqs)]
    lens = [n + 9 if n else 0 for n in all_news]
    case = Pool(cuda, fmt, 64, 1, 64, lens, rng)
    case.fill_at_once(rng)
    case.upload()
    q = (rng.standard_normal((sum(all_news) + 1, 4 * 64)) * 1.5).astype(np.float32)
    got = attend(cuda, case, all_news, 4, q, rows=case.rows(all_news, n_rows=q.shape[0], max_queries=hint))
    with_rows = sorted(news)
    case.table, case.lens = case.table[with_rows], [lens[s] for s in with_rows]
    check(case, [news[s] for s in with_rows], 4, q, got)


@pytest.mark.parametrize("fmt", [F16, I8])
@pytest.mark.parametrize("hint", [1, 1000])
def test_chunks_among_thousands_of_single_tokens(cuda, hint, fmt):
    n_seqs = 3000
    rng = np.random.default_rng(91)
    news = [150 if s in (0, 1500, 2999) else 1 for s in range(n_seqs)]
    lens = [n + int(rng.integers(0, 40)) for n in news]
    case = Pool(cuda, fmt, 16, 1, 64, lens, rng)
    case.fill_at_once(rng)
    case.upload()
    q = (rng.standard_normal((sum(news), 2 * 64)) * 1.5).astype(np.float32)
    check(case, news, 2, q, attend(cuda, case, news, 2, q, rows=case.rows(news, max_queries=hint)))
