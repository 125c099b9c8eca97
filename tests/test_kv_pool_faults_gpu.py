"""A page that the pool does not have is reported by the wait for the recording that met it, and by no other: not another recording's, not another
backend's, not a model's step. A captured call's is reported by its backend's next wait."""

import numpy as np
import pytest

from bobcat_b200 import Cuda, F16, KvRows, Lfm2Cuda, Model, errors
from kv_pool_cases import Pool

pytestmark = pytest.mark.gpu

HD = 64


class Calls:
    """A pool on a backend of its own, and attention over it with a table that is right and one that is not."""

    def __init__(self, stream=None):
        self.cuda = Cuda.open(0, stream)
        self.case = Pool(self.cuda, F16, 16, 1, HD, [40], np.random.default_rng(1))
        self.case.fill(np.random.default_rng(2))
        self.case.upload()
        self.rows = {"good": self.case.rows([1])}
        self.case.table[0, 1] = self.case.n_pages + 7
        self.rows["bad"] = self.case.rows([1])
        self.case.lens = [49]
        self.rows["long"] = KvRows(1, 1, 1, 3, *(self.rows["good"].holds[:2]), self.cuda.buffer_from(np.array([49], dtype=np.uint32)))
        self.q, self.out = self.cuda.new_buffer(HD * 4), self.cuda.new_buffer(HD * 4)
        self.scratch = self.cuda.new_buffer(4 * self.cuda.attention_paged_scratch_floats(1, 1, HD))

    def attend(self, which):
        self.cuda.attention_paged(self.case.pool, self.rows[which], self.q, self.scratch, self.out, 1, HD, HD)

    def commit(self, which):
        self.cuda.begin()
        self.attend(which)
        return self.cuda.commit()


@pytest.fixture
def two():
    calls = [Calls(), Calls()]
    yield calls
    for c in calls:
        c.cuda.close()


def settle():
    torch = pytest.importorskip("torch")
    torch.cuda.synchronize()


def test_another_backend_is_not_blamed(two):
    a, b = two
    ticket = a.commit("bad")
    settle()  # whatever a's kernels leave behind is there
    b.cuda.wait(b.commit("good"))
    with pytest.raises(errors.OutOfBounds, match="page"):
        a.cuda.wait(ticket)
    a.cuda.wait(a.commit("good"))  # reported once


def test_each_backend_learns_of_its_own(two):
    tickets = [c.commit("bad") for c in two]
    settle()
    for c, t in zip(two, tickets):
        with pytest.raises(errors.OutOfBounds, match="page"):
            c.cuda.wait(t)


def test_another_recording_is_not_blamed(two):
    a = two[0]
    tickets = [a.commit(w) for w in ("good", "bad", "good", "long", "good")]
    settle()
    for i in (4, 0, 2):
        a.cuda.wait(tickets[i])
    with pytest.raises(errors.OutOfBounds, match="positions"):
        a.cuda.wait(tickets[3])
    with pytest.raises(errors.OutOfBounds, match="page"):
        a.cuda.wait(tickets[1])
    for t in tickets:
        a.cuda.wait(t)  # collected


def test_a_discarded_recording_blames_nobody(two):
    a = two[0]
    a.cuda.begin()
    a.attend("bad")
    a.cuda.discard()
    a.cuda.wait(a.commit("good"))


def test_a_model_is_not_blamed(two, model_path):
    a = two[0]
    path = model_path("lfm2-small")
    cuda = Cuda.open(0)
    try:
        seq = Lfm2Cuda(Model.load(path), cuda, 64, kv_half=False)
        seq.prefill(np.arange(1, 9, dtype=np.uint32))
        ticket = a.commit("bad")
        settle()
        assert len(seq.generate(3)) == 3
        with pytest.raises(errors.OutOfBounds):
            a.cuda.wait(ticket)
        seq.close()
    finally:
        cuda.close()


def test_many_recordings_before_any_wait(two):
    """More than the words that a device has at first."""
    a = two[0]
    tickets = [a.commit("bad" if i % 3 == 0 else "good") for i in range(1500)]
    for i, t in enumerate(tickets):
        if i % 3 == 0:
            with pytest.raises(errors.OutOfBounds):
                a.cuda.wait(t)
        else:
            a.cuda.wait(t)


def test_a_captured_call_is_reported_by_its_backends_next_wait():
    torch = pytest.importorskip("torch")
    stream = torch.cuda.Stream()
    a, b = Calls(stream.cuda_stream), Calls()
    graph = torch.cuda.CUDAGraph()
    a.cuda.wait(a.commit("good"))
    a.cuda.begin()
    with torch.cuda.graph(graph, stream=stream):
        a.attend("bad")
    a.cuda.end()  # recorded, not run
    for _ in range(2):
        with torch.cuda.stream(stream):
            graph.replay()
        settle()
        b.cuda.wait(b.commit("good"))
        with pytest.raises(errors.OutOfBounds, match="page"):
            a.cuda.wait(a.commit("good"))
        a.cuda.wait(a.commit("good"))
    del graph
    a.cuda.close()
    b.cuda.close()
