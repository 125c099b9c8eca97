"""The pool's and the rows' buffers are named when a call is made, as those of every other op: one that was freed meanwhile reaches the library as no
buffer, which it refuses, and not as the address of a handle that is gone."""

import ctypes as C

import pytest

from bobcat_b200 import I8, Buffer, Cuda, KvPool, KvRows


class Library:
    """Notes the handles of a call; frees are taken."""

    def __init__(self):
        self.seen = None

    def bc_buffer_free(self, handle):
        pass

    def _op(self, backend, pool, rows, *rest):
        self.seen = dict(k=(pool.k, pool.k_off), v=(pool.v, pool.v_off), table=(rows.table, rows.table_off), starts=(rows.starts, rows.starts_off),
                         lens=(rows.lens, rows.lens_off))
        return 0

    bc_op_kv_write = bc_op_kv_read = bc_op_attention_paged = _op


@pytest.fixture
def fake():
    cuda = object.__new__(Cuda)
    cuda._L, cuda._h = Library(), None
    buffers = {name: Buffer(cuda, C.c_void_p(0x1000 * (i + 1))) for i, name in enumerate(("k", "v", "table", "starts", "lens"))}
    pool = KvPool(I8, 4, 16, 2, 64, buffers["k"], buffers["v"].at(256))
    rows = KvRows(1, 5, 5, 2, buffers["table"].at(8), buffers["starts"], buffers["lens"].at(4))
    calls = [lambda: cuda.kv_write(pool, rows, None, None, 128, 128), lambda: cuda.kv_read(pool, rows, None, None, False, 128, 128),
             lambda: cuda.attention_paged(pool, rows, None, None, None, 2, 128, 64)]
    return cuda, buffers, calls


def test_handles_and_offsets(fake):
    cuda, _, calls = fake
    for call in calls:
        call()
        assert cuda._L.seen == dict(k=(0x1000, 0), v=(0x2000, 256), table=(0x3000, 8), starts=(0x4000, 0), lens=(0x5000, 4))


@pytest.mark.parametrize("name", ["k", "v", "table", "starts", "lens"])
def test_a_freed_buffer_is_no_buffer(fake, name):
    cuda, buffers, calls = fake
    buffers[name].free()
    for call in calls:
        call()
        assert cuda._L.seen[name][0] is None
        assert all(handle is not None for other, (handle, _) in cuda._L.seen.items() if other != name)
