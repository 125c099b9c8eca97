"""Refusals of calls over the key/value pool that would read or write what is not theirs: buffers longer than the memory under them, results over queries or
scratch."""

import numpy as np
import pytest

from bobcat_b200 import F16, errors
from kv_pool_cases import Pool

pytestmark = pytest.mark.gpu


def test_a_buffer_ends_with_the_memory_under_it(cuda):
    torch = pytest.importorskip("torch")
    size = 64 << 20
    t = torch.zeros(size, dtype=torch.uint8, device="cuda")
    for n in (1, 256, size):
        cuda.buffer_at(t.data_ptr(), n).free()
    cuda.buffer_at(t.data_ptr() + 256, size - 256).free()
    base, reserved = 0, 0
    for segment in torch.cuda.memory_snapshot():
        if segment["address"] <= t.data_ptr() < segment["address"] + segment["total_size"]:
            base, reserved = segment["address"], segment["total_size"]
    assert reserved >= size
    cuda.buffer_at(base, reserved).free()
    for n in (reserved + 1, reserved + (1 << 20), 1 << 45, (1 << 64) - 256):
        with pytest.raises(errors.Argument, match="bytes"):
            cuda.buffer_at(base, n)
    with pytest.raises(errors.Argument):
        cuda.buffer_at(base + 256, reserved - 255)
    own = cuda.new_buffer(8 << 20)
    cuda.buffer_at(own.device_ptr, 8 << 20).free()
    with pytest.raises(errors.Argument):
        cuda.buffer_at(own.device_ptr, 1 << 40)


def test_results_over_queries_or_scratch(cuda):
    kv, hd, heads, n = 2, 64, 4, 5
    case = Pool(cuda, F16, 16, kv, hd, [20], np.random.default_rng(80))
    case.fill(np.random.default_rng(81))
    pool, rows = case.upload(), case.rows([n])
    width, need = heads * hd, cuda.attention_paged_scratch_floats(heads, kv, hd)
    big = cuda.new_buffer(4 * (need + 64 * width))
    q, out, scratch = cuda.new_buffer(4 * n * width), cuda.new_buffer(4 * n * width), cuda.new_buffer(4 * need)
    wide = 3 * width  # rows of a product: queries, keys, values
    at = big.floats

    def refused(q, scratch, out, stride=width, head_stride=hd):
        with pytest.raises(errors.Argument, match="overlap"):
            cuda.attention_paged(pool, rows, q, scratch, out, heads, stride, head_stride)

    cuda.begin()
    try:
        refused(q, scratch, q)
        refused(at(0), scratch, at(4))
        refused(at(4), scratch, at(0))
        refused(at(0), scratch, at((n - 1) * wide), stride=wide)               # over the last row
        refused(at(0), scratch, at(456), stride=40 * width, head_stride=132)    # a row's last head ends at 3 * 132 + 64 = 460
        refused(at(0), at((n - 1) * width), out)
        refused(at(need), at(0 + 4), out)
        refused(q, at(0), at(need - 4))
        refused(q, at(4), at(0))
        refused(q, q if need <= n * width else at(0), at(0))
        t = cuda.buffer_at(big.device_ptr, 4 * (need + 64 * width))            # the same memory under another handle
        refused(at(0), scratch, t.floats(4))
        refused(t.floats(0), scratch, at(n * width - 4))
        # Beside one another in one buffer, and in what rows leave between them.
        cuda.attention_paged(pool, rows, at(0), at(2 * n * width), at(n * width), heads, width, hd)
        cuda.attention_paged(pool, rows, at(0), scratch, at(width), heads, 8 * width, hd)
        cuda.attention_paged(pool, rows, at(0), scratch, at(460), heads, 10 * width, 132)
        cuda.end()
    except BaseException:
        cuda.discard()
        raise
