"""The serving loop when a step fails, without a GPU: the model's forward is a stand-in, the cache
the host bookkeeping alone.  What a failed call took is given back."""
import pytest
import torch

from src import paged_kv_cache
from src.paged_kv_cache import OutOfPages, PageAllocator, PagedKVCache
from src.paged_llama import PagedLlama


class Broken(RuntimeError):
    pass


class Cache(PageAllocator):
    def extend(self, seqs, counts):
        super().extend(seqs, counts)
        return len(seqs)


def make(num_pages, page_size, fails=()):
    """A server whose forward raises at the calls numbered in `fails`."""
    server = PagedLlama.__new__(PagedLlama)
    server.cache = Cache(num_pages, page_size)
    server.calls = 0

    def forward(step, tokens, prompt):
        server.calls += 1
        if server.calls in fails:
            raise Broken("forward")
        return torch.zeros(step, 10)

    server._forward = forward
    return server


def test_generate_gives_its_pages_back():
    server = make(4, 4)
    kept = server.cache.new_sequence()
    with pytest.raises(OutOfPages):
        server.generate([[1] * 6, [2] * 6], 8)  # two pages each, and a third for the ninth token
    assert server.cache.free_pages == 4 and server.cache.sequences() == [kept]
    assert server.generate([[1] * 6], 3) == [[0, 0, 0]]
    assert server.cache.free_pages == 4 and server.cache.sequences() == [kept]


@pytest.mark.parametrize("call", [1, 2, 3])
def test_a_failing_forward_gives_its_pages_back(call):
    server = make(8, 4, fails=(call,))
    with pytest.raises(Broken):
        server.generate([[1] * 6, [2] * 3], 4)
    assert server.cache.free_pages == 8 and server.cache.sequences() == []


def test_a_failing_prefill_leaves_the_others():
    server = make(8, 4, fails=(2,))
    seqs, _ = server.prefill([[1, 2, 3]])
    with pytest.raises(Broken):
        server.prefill([[4] * 9, [5]])
    assert server.cache.sequences() == seqs and server.cache.free_pages == 7


def test_a_failing_decode_can_be_repeated():
    server = make(8, 4, fails=(2,))
    seqs, _ = server.prefill([[1] * 4, [2] * 3])
    fork = server.cache.fork(seqs[1])
    before = [server.cache.length(s) for s in seqs + [fork]], server.cache.free_pages
    with pytest.raises(Broken):
        server.decode(seqs, [5, 6])
    assert [server.cache.length(s) for s in seqs + [fork]] == before[0]
    # The page that seqs[1] shared has been copied for it; a page of no token is not kept.
    assert server.cache.free_pages == before[1] - 1
    assert server.decode(seqs, [5, 6]).shape == (2, 10)
    assert [server.cache.length(s) for s in seqs + [fork]] == [5, 4, 3]
    for s in seqs + [fork]:
        server.cache.free(s)
    assert server.cache.free_pages == 8


def test_withdraw():
    a = PageAllocator(10, 4)
    s, t = a.new_sequence(), a.new_sequence()
    a.extend([s, t], [9, 4])
    for n, pages in ((0, 3), (1, 2), (3, 2), (1, 1), (4, 0)):
        a.withdraw([s], [n])
        assert len(a.pages(s)) == pages == -(-a.length(s) // 4)
    assert a.length(s) == 0 and a.free_pages == 9
    a.extend([s], [5])
    f = a.fork(s)
    a.withdraw([s, t], [5, 0])
    assert a.length(f) == 5 and len(a.pages(f)) == 2 and a.free_pages == 7
    with pytest.raises(ValueError, match="5 tokens of a sequence of 4"):
        a.withdraw([f, t], [1, 5])
    with pytest.raises(ValueError, match="one count"):
        a.withdraw([t, t], [1, 1])
    with pytest.raises(KeyError, match="no sequence"):
        a.withdraw([99], [1])
    assert a.length(f) == 5 and a.length(t) == 4


def test_a_step_without_memory_is_taken_back(monkeypatch):
    cache = PagedKVCache(1, 8, 4, 1, 64, device="cpu")
    s = cache.new_sequence()
    cache.extend([s], [3])

    def no_memory(*args, **kwargs):
        raise MemoryError("step")

    with monkeypatch.context() as m:
        m.setattr(paged_kv_cache.torch, "tensor", no_memory)
        with pytest.raises(MemoryError):
            cache.extend([s], [9])
    assert cache.length(s) == 3 and cache.free_pages == 7
    step = cache.extend([s], [9])
    assert step.start_lens.tolist() == [3] and step.seq_lens.tolist() == [12]
    assert step.positions.tolist() == list(range(3, 12)) and not step.fresh
