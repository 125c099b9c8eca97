"""Keys of half pages that hold infinities (what kv_write stores of elements above 65 504): a score of minus infinity weighs nothing, as by the formula; one of
plus infinity, or of no number, leaves its row no number."""

import numpy as np
import pytest

from bobcat_b200 import F16
from kv_pool_cases import Pool, attention
from test_attention_paged_gpu import MARK, attend, build

pytestmark = pytest.mark.gpu

INF, NAN = np.inf, np.nan


@pytest.mark.parametrize("hint", [1, 1000])
@pytest.mark.parametrize("heads, kv, hd", [(8, 2, 64), (7, 1, 64), (4, 2, 128), (8, 1, 128), (3, 1, 256), (8, 1, 256)])
@pytest.mark.parametrize("at", [0, 40, 70])
def test_infinite_keys(cuda, at, heads, kv, hd, hint):
    first, length, group = 8, 140, heads // kv
    n = length - first
    case = build(cuda, F16, 16, kv, hd, [length], seed=60)
    rng = np.random.default_rng(61)
    special = []
    for i, elements in enumerate([{5: INF}, {9: -INF}, {5: INF, 9: -INF}, {33: INF}]):
        key = rng.standard_normal((kv, hd)).astype(np.float32)
        for e, x in elements.items():
            key[:, e] = x
        special.append((at + 7 * i, key))
    for pos, key in special:
        case.put(case.k_raw, 0, pos, key)
    case.upload()
    q = np.random.default_rng(62).standard_normal((n, heads, hd)).astype(np.float32) * 1.5
    # Most rows' scores with all of these are minus infinity; some elements are zero, or too small to be halves beside their rows' largest.
    sign = np.where(np.random.default_rng(63).random((n, heads)) < 0.8, 1.0, -1.0)
    q[..., 5] = -np.abs(q[..., 5]) * sign
    q[..., 9] = np.abs(q[..., 9])
    q[..., 33] = -1e-30
    q[20:30, :, 33] = 0.0
    q = q.astype(np.float32)
    got = attend(cuda, case, [n], heads, q.reshape(n, -1), rows=case.rows([n], max_queries=hint)).reshape(n, heads, hd)
    k, v = case.context(case.k_raw, 0, length), case.context(case.v_raw, 0, length)
    positions = [pos for pos, _ in special]
    finite = 0
    for h in range(heads):
        with np.errstate(invalid="ignore"):
            s = (q[:, h].astype(np.float64)[:, None] * k[None, positions, h // group]).sum(-1)
        for i in range(n):
            seen = [j for j, pos in enumerate(positions) if pos <= first + i]
            have = got[i, h]
            if any(not (s[i, j] == -INF) for j in seen):
                assert np.isnan(have).all(), (i, h)
                continue
            keep = np.array([p for p in range(first + i + 1) if p not in positions])
            one = attention(q[i:i + 1, h:h + 1], k[keep, h // group:h // group + 1], v[keep, h // group:h // group + 1], len(keep) - 1)
            assert (np.abs(have - one[0][0, 0]) <= one[1][0, 0]).all(), (i, h)
            finite += len(seen) > 0
    assert finite > n * heads // 8


@pytest.mark.parametrize("hint", [1, 1000])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_a_key_that_is_no_number_and_rows_all_of_whose_scores_are_minus_infinity(cuda, hd, hint):
    case = build(cuda, F16, 32, 1, hd, [200], seed=64)
    key = np.ones((1, hd), dtype=np.float32)
    key[0, 3] = INF
    for pos in range(3):
        case.put(case.k_raw, 0, pos, key)
    key[0, 3] = NAN
    case.put(case.k_raw, 0, 150, key)
    case.upload()
    q = np.random.default_rng(65).standard_normal((200, 2 * hd)).astype(np.float32)
    q[:, 3] = q[:, hd + 3] = -1.0
    got = attend(cuda, case, [200], 2, q, rows=case.rows([200], max_queries=hint)).reshape(200, 2, hd)
    assert (got[:3] == 0).all()  # they see keys that weigh nothing
    k, v = case.context(case.k_raw, 0, 150)[3:], case.context(case.v_raw, 0, 150)[3:]
    want, bound = attention(q[3:150].reshape(147, 2, hd), k, v, 0)
    assert (np.abs(got[3:150] - want) <= bound).all()
    assert np.isnan(got[150:]).all()


@pytest.mark.parametrize("hint", [1, 1000])
@pytest.mark.parametrize("heads, kv, hd", [(16, 8, 64), (8, 8, 128), (14, 2, 256)])
def test_infinite_keys_of_long_contexts(cuda, heads, kv, hd, hint):
    """Row tiles over many CTAs and whole ones, beside single tokens: what the contexts hold ahead of the rows weighs nothing on any of them."""
    rng = np.random.default_rng(66)
    news, lens = [70, 1, 300, 2, 33], [6000, 4000, 310, 900, 2500]
    special = [[3, 127, 128, 5000], [64], [2], [0, 800], [31, 1000, 2000]]
    case = Pool(cuda, F16, 64, kv, hd, lens, rng)
    case.fill_at_once(rng)
    for s, positions in enumerate(special):
        for pos in positions:
            key = rng.standard_normal((kv, hd)).astype(np.float32)
            key[:, 7] = INF
            case.put(case.k_raw, s, pos, key)
    case.upload()
    q = (rng.standard_normal((sum(news) + 1, heads, hd)) * 1.5).astype(np.float32)
    q[..., 7] = -np.abs(q[..., 7])
    got = attend(cuda, case, news, heads, q.reshape(len(q), -1), rows=case.rows(news, n_rows=len(q), max_queries=hint)).reshape(len(q), heads, hd)
    at = 0
    for s, n in enumerate(news):
        k, v = (np.delete(case.context(raw, s, lens[s]), special[s], axis=0) for raw in (case.k_raw, case.v_raw))
        want, bound = attention(q[at:at + n], k, v, lens[s] - n - len(special[s]))
        assert (np.abs(got[at:at + n] - want) <= bound).all(), s
        at += n
    assert (got[at:] == MARK).all()
