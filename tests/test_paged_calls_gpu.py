"""Refusals of calls over the key/value pool that would read or write what is not theirs: buffers longer than the memory under them."""

import pytest

from bobcat_b200 import errors

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
