"""Attention over pages of numbers far apart: 8-bit value rows of very different scales within a key tile. Against 64 bits, within the bound
of kv_pool_cases.attention and the floor of 8-bit values' weights."""

import numpy as np
import pytest

from bobcat_b200 import I8
from kv_pool_cases import Pool, attention
from test_attention_paged_gpu import attend, build

pytestmark = pytest.mark.gpu

SHAPES = [(64, 2, 8), (128, 2, 4), (256, 1, 2), (64, 1, 7)]


def floor_of_weights(case, q, first, length):
    """How far 8-bit values' weights may take an answer off beside their 22 bits, [n][heads][hd].

    A weight, probability p times scale d, is two halves in a unit that makes the row's largest weight W, of the positions that it sees, 2^7 at the
    least (128 scales at most to one weight, 2^14 units to a scale; 2^11 in the kernel of single tokens). Halves end in steps of 2^-24, so each
    weight is off by 2^-25 units, 2^-32 W, and an element by that times the sum of its whole numbers, over the sum of probabilities."""
    n, heads, hd = q.shape
    group, m = heads // case.kv, case.kv * case.page_size * case.row_bytes
    pos = np.arange(length)
    page, slot = case.table[0, pos // case.page_size], pos % case.page_size
    whole = case.v_raw[:, :m].reshape(case.n_pages, case.kv, case.page_size, case.row_bytes)[page, :, slot].astype(np.float64) - 128.0
    d = np.ascontiguousarray(case.v_raw[:, m:].reshape(case.n_pages, case.kv, case.page_size, 4)[page, :, slot]).view(np.float32).reshape(length, case.kv).astype(np.float64)
    k = case.context(case.k_raw, 0, length)
    out = np.zeros((n, heads, hd))
    for h in range(heads):
        s = q[:, h].astype(np.float64) @ k[:, h // group].T / np.sqrt(hd)
        s[np.arange(length) > first + np.arange(n)[:, None]] = -np.inf
        p = np.exp(s - s.max(axis=1, keepdims=True))
        seen = np.isfinite(s).astype(np.float64)
        heaviest = (p * d[:, h // group]).max(axis=1, keepdims=True)
        out[:, h] = 2.0 ** -32 * heaviest * (seen @ np.abs(whole[:, h // group])) / p.sum(axis=1, keepdims=True)
    return out


def within(case, got, q, first, heads, length):
    q, hd = q.reshape(-1, heads, case.hd), case.hd
    want, bound = attention(q, case.context(case.k_raw, 0, length), case.context(case.v_raw, 0, length), first)
    bound = bound + floor_of_weights(case, q, first, length)
    have = got.reshape(-1, heads, hd)
    assert np.isfinite(have).all()
    assert (np.abs(have - want) <= bound).all(), (np.abs(have - want) / np.maximum(bound, 1e-300)).max()


@pytest.mark.parametrize("hint", [1, 1000])
@pytest.mark.parametrize("hd, kv, heads", SHAPES)
@pytest.mark.parametrize("ratio", [1e3, 1e6, 1e8, 1e10, 1e12, 1e20])
def test_large_values_of_a_later_position_leave_earlier_rows_alone(cuda, ratio, hd, kv, heads, hint):
    """Position 60 of 100 holds values `ratio` times the others', in the same key tile as those of the rows before it, which do not see it; rows behind it
    do."""
    case = build(cuda, I8, 16, kv, hd, [100], seed=50)
    rng = np.random.default_rng(51)
    case.put(case.v_raw, 0, 60, (rng.standard_normal((kv, hd)) * ratio).astype(np.float32))
    case.upload()
    q = (rng.standard_normal((90, heads * hd)) * 1.5).astype(np.float32)
    got = attend(cuda, case, [90], heads, q, rows=case.rows([90], max_queries=hint))
    within(case, got[:50], q[:50], 10, heads, 60)  # positions 10 .. 59
    within(case, got, q, 10, heads, 100)


@pytest.mark.parametrize("hint", [1, 1000])
@pytest.mark.parametrize("scale", [1e30, 2.5e36])
def test_the_largest_values_and_keys_of_a_later_position_leave_earlier_rows_alone(cuda, scale, hint):
    """As large as 8-bit rows can be: no product of theirs gets into rows that do not see them."""
    kv, hd, heads = 2, 64, 8
    case = build(cuda, I8, 16, kv, hd, [100], seed=52)
    rng = np.random.default_rng(53)
    for raw in (case.k_raw, case.v_raw):
        case.put(raw, 0, 60, np.full((kv, hd), scale * 127, dtype=np.float32))
    case.upload()
    q = (rng.standard_normal((50, heads * hd)) * 1.5).astype(np.float32)
    got = attend(cuda, case, [50], heads, q, rows=case.rows([50], lens=[60], max_queries=hint))  # the same rows, of a shorter sequence
    within(case, got, q, 10, heads, 60)
    longer = np.concatenate([q, np.zeros((40, heads * hd), dtype=np.float32)])
    got = attend(cuda, case, [90], heads, longer, rows=case.rows([90], max_queries=hint))
    within(case, got[:50], q, 10, heads, 60)


@pytest.mark.parametrize("hint", [1, 1000])
@pytest.mark.parametrize("hd, kv, heads", SHAPES)
@pytest.mark.parametrize("ratio", [1e6, 1e10, 1e15])
@pytest.mark.parametrize("weight", [1e-4, 1e-9, 1e-14, 1e-25])
def test_large_values_of_a_position_that_hardly_counts(cuda, weight, ratio, hd, kv, heads, hint):
    """Position 60's probability is about `weight` of the others', its values are `ratio` times theirs: its share may be everything, as much as theirs, or
    nothing to speak of, and theirs keeps its bits where it counts."""
    case = build(cuda, I8, 32, kv, hd, [300], seed=54)
    rng = np.random.default_rng(55)
    at, gap = 60, -np.log(weight)
    key = (rng.standard_normal((kv, hd)) * 0.1).astype(np.float32)
    key[:, 0] = -gap * np.sqrt(hd) / 8.0
    case.put(case.k_raw, 0, at, key)
    case.put(case.v_raw, 0, at, (rng.standard_normal((kv, hd)) * ratio).astype(np.float32))
    case.upload()
    q = rng.standard_normal((280, heads * hd)).astype(np.float32)
    q.reshape(280, heads, hd)[:, :, 0] = 8.0
    within(case, attend(cuda, case, [280], heads, q, rows=case.rows([280], max_queries=hint)), q, 20, heads, 300)


@pytest.mark.parametrize("hint", [1, 1000])
@pytest.mark.parametrize("hd, kv, heads", SHAPES)
def test_value_rows_of_zeros_and_of_every_size(cuda, hd, kv, heads, hint):
    """Scales 2^12 apart from position to position, many of them zero, whole key tiles of zeros among them."""
    case = Pool(cuda, I8, 16, kv, hd, [700], np.random.default_rng(56))
    rng = np.random.default_rng(57)
    for pos in range(700):
        size = 0.0 if pos % 3 == 0 or 128 <= pos < 300 or pos < 20 else 2.0 ** rng.integers(-60, 60)
        case.put(case.k_raw, 0, pos, rng.standard_normal((kv, hd)).astype(np.float32))
        case.put(case.v_raw, 0, pos, (rng.standard_normal((kv, hd)) * size).astype(np.float32))
    case.upload()
    q = (rng.standard_normal((695, heads * hd)) * 1.5).astype(np.float32)
    within(case, attend(cuda, case, [695], heads, q, rows=case.rows([695], max_queries=hint)), q, 5, heads, 700)


@pytest.mark.parametrize("hint", [1, 1000])
@pytest.mark.parametrize("hd, kv, heads", SHAPES)
@pytest.mark.parametrize("gap", [0.0, 8.0, 25.0])
def test_a_first_position_of_small_values(cuda, gap, hd, kv, heads, hint):
    """What prompts begin with often has small values and takes most of the probability, of some heads' queries: the others' share is what the rows are about, in
    every tile behind it."""
    case = build(cuda, I8, 32, kv, hd, [1500], seed=58)
    rng = np.random.default_rng(59)
    key = (rng.standard_normal((kv, hd)) * 0.1).astype(np.float32)
    key[:, 0] = gap * np.sqrt(hd) / 4.0
    case.put(case.k_raw, 0, 0, key)
    case.put(case.v_raw, 0, 0, (rng.standard_normal((kv, hd)) * 1e-6).astype(np.float32))
    case.put(case.v_raw, 0, 700, (rng.standard_normal((kv, hd)) * 1e7).astype(np.float32))
    case.upload()
    q = rng.standard_normal((300, heads, hd)).astype(np.float32)
    q[:, ::2, 0] = 4.0
    within(case, attend(cuda, case, [300], heads, q.reshape(300, -1), rows=case.rows([300], max_queries=hint)), q, 1200, heads, 1500)
