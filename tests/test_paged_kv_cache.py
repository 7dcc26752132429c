"""Host bookkeeping of the paged cache (no GPU): growth, sharing, copy on
write, freeing and compaction, against a model that follows the contents of
every page; and the refusals of the serving entry points of the C ABI."""
import random

import pytest

from src import capi
from src.paged_kv_cache import OutOfPages, PageAllocator


class Contents:
    """What the pages would hold: (page, slot) -> token."""

    def __init__(self, alloc):
        self.alloc, self.mem, self.want, self.tokens = alloc, {}, {}, 0

    def move(self, moves):
        assert len({b for _, b in moves}) == len(moves)
        assert not {a for a, _ in moves} & {b for _, b in moves}
        size = self.alloc.page_size
        for a, b in moves:
            for s in range(size):
                self.mem[b, s] = self.mem.get((a, s))

    def extend(self, seqs, counts):
        self.move(self.alloc.extend(seqs, counts))
        for seq, n in zip(seqs, counts):
            for _ in range(n):
                at = len(self.want[seq])
                page = self.alloc.pages(seq)[at // self.alloc.page_size]
                self.mem[page, at % self.alloc.page_size] = self.tokens
                self.want[seq].append(self.tokens)
                self.tokens += 1

    def check(self):
        a, size = self.alloc, self.alloc.page_size
        used = set()
        for seq, want in self.want.items():
            pages = a.pages(seq)
            assert a.length(seq) == len(want) and len(pages) == -(-len(want) // size)
            assert [self.mem[pages[t // size], t % size] for t in range(len(want))] == want
            used |= set(pages)
        assert a.free_pages == a.num_pages - len(used)
        assert not used & set(a._free)


@pytest.mark.parametrize("seed", range(8))
def test_random_histories(seed):
    rng = random.Random(seed)
    alloc = PageAllocator(rng.choice([6, 40, 150]), rng.choice([1, 4, 16]))
    c = Contents(alloc)
    for _ in range(300):
        live = list(c.want)
        op = rng.random()
        if op < 0.2 or not live:
            c.want[alloc.new_sequence()] = []
        elif op < 0.35:
            seq = rng.choice(live)
            c.want[alloc.fork(seq)] = list(c.want[seq])
        elif op < 0.45:
            seq = rng.choice(live)
            alloc.free(seq)
            del c.want[seq]
        elif op < 0.5:
            c.move(alloc.compact())
            used = {p for s in c.want for p in alloc.pages(s)}
            assert used == set(range(len(used)))
        else:
            seqs = rng.sample(live, rng.randint(1, len(live)))
            counts = [rng.choice([0, 1, 1, 1, 5, 20]) for _ in seqs]
            before = ({s: alloc.pages(s) for s in live}, alloc.free_pages)
            try:
                c.extend(seqs, counts)
            except OutOfPages:
                assert before == ({s: alloc.pages(s) for s in live}, alloc.free_pages)
        c.check()


def test_forks_share_until_one_writes():
    a = PageAllocator(10, 4)
    s = a.new_sequence()
    assert a.extend([s], [6]) == []
    f = a.fork(s)
    assert a.pages(f) == a.pages(s) and a.free_pages == 8
    # Both write in one step: one copies, the other keeps the page.
    moves = a.extend([s, f], [1, 1])
    assert len(moves) == 1 and moves[0][0] == a.pages(f)[1] and moves[0][1] == a.pages(s)[1]
    assert a.pages(s)[0] == a.pages(f)[0] and a.free_pages == 7
    # A full last page is not written to again: nothing is copied.
    a.extend([s, f], [1, 1])
    g = a.fork(s)
    assert a.extend([g], [1]) == []
    a.free(s)
    a.free(f)
    a.free(g)
    assert a.free_pages == 10


def test_allocator_refusals():
    with pytest.raises(ValueError, match="positive"):
        PageAllocator(0, 16)
    a = PageAllocator(4, 4)
    s = a.new_sequence()
    with pytest.raises(OutOfPages, match="5 pages are needed, 4 of 4"):
        a.extend([s], [17])
    assert a.length(s) == 0 and a.free_pages == 4
    with pytest.raises(ValueError, match="once a step"):
        a.extend([s, s], [1, 1])
    with pytest.raises(ValueError, match="negative"):
        a.extend([s], [-1])
    with pytest.raises(ValueError, match="same length"):
        a.extend([s], [1, 2])
    for call in (lambda: a.extend([7], [1]), lambda: a.fork(7), lambda: a.free(7),
                 lambda: a.pages(7), lambda: a.length(7)):
        with pytest.raises(KeyError, match="no sequence 7"):
            call()


# ------------------------------------------------- C ABI, refused on the host


def prompt(dtype=capi.FRN_DTYPE_BF16, ptr=16, qs=(1024, 128), ks=(256, 128), vs=(256, 128),
           os_=(1024, 128), cu=16, batch=1, tokens=4, longest=4, Hq=8, Hkv=2, D=128, Dv=128):
    return capi.lib().frn_gqa_prompt_attention(dtype, ptr, *qs, 16, *ks, 16, *vs, 16, *os_, cu,
                                               batch, tokens, longest, Hq, Hkv, D, Dv, 0.1, None)


@pytest.mark.parametrize("kwargs,code", [
    (dict(dtype=capi.FRN_DTYPE_F32), capi.FRN_ERR_UNSUPPORTED),
    (dict(D=96, Dv=96), capi.FRN_ERR_UNSUPPORTED),
    (dict(D=128, Dv=64), capi.FRN_ERR_UNSUPPORTED),
    (dict(Hq=9), capi.FRN_ERR_UNSUPPORTED),
    (dict(Hq=258), capi.FRN_ERR_UNSUPPORTED),
    (dict(Hkv=0), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(batch=-1), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(tokens=-4), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(tokens=1 << 31), capi.FRN_ERR_UNSUPPORTED),
    (dict(ptr=None), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(cu=None), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(ptr=24), capi.FRN_ERR_MISALIGNED),
    (dict(qs=(1024, 132)), capi.FRN_ERR_MISALIGNED),
    (dict(ks=(64, 128)), capi.FRN_ERR_MISALIGNED),
    (dict(vs=(256, 0)), capi.FRN_ERR_MISALIGNED),
    (dict(os_=(1024, -128)), capi.FRN_ERR_MISALIGNED),
])
def test_prompt_attention_refusals(kwargs, code):
    assert prompt(**kwargs) == code
    assert capi.last_error() != ""


def test_prompt_attention_of_nothing():
    assert prompt(batch=0, ptr=None) == capi.FRN_OK
    assert prompt(tokens=0, ptr=None, cu=None) == capi.FRN_OK


def cache(**kw):
    fields = dict(k=16, v=16, num_pages=4, page_size=16, num_kv_heads=2, head_dim=128,
                  k_page_stride=4096, k_token_stride=256, k_head_stride=128, v_page_stride=4096,
                  v_token_stride=256, v_head_stride=128, page_table=16, page_table_stride=8,
                  max_pages=8)
    fields.update(kw)
    return capi.PagedKV(**fields)


BAD_CACHES = [
    (dict(page_size=0), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(num_kv_heads=-1), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(head_dim=80), capi.FRN_ERR_UNSUPPORTED),
    (dict(k=None), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(v=40), capi.FRN_ERR_MISALIGNED),
    (dict(page_table=None), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(page_table_stride=7), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(k_token_stride=252), capi.FRN_ERR_MISALIGNED),
    (dict(v_head_stride=64), capi.FRN_ERR_MISALIGNED),
    (dict(max_pages=1 << 28, page_table_stride=1 << 28), capi.FRN_ERR_UNSUPPORTED),
]


def decode(c, dtype=capi.FRN_DTYPE_BF16, q=16, qs=(1024, 128), lens=16, batch=1, Hq=8, ws=16,
           ws_bytes=1 << 20):
    import ctypes
    return capi.lib().frn_gqa_paged_decode_attention(
        dtype, q, *qs, ctypes.byref(c) if c is not None else None, lens, 16, 1024, 128, batch, Hq,
        0.1, ws, ws_bytes, None)


def append(c, dtype=capi.FRN_DTYPE_BF16, k=16, ks=(256, 128), start=16, cu=None, batch=2, tokens=2):
    import ctypes
    return capi.lib().frn_kv_cache_append(
        dtype, k, *ks, 16, 256, 128, ctypes.byref(c) if c is not None else None, start, cu, batch,
        tokens, None)


@pytest.mark.parametrize("call", [decode, append])
@pytest.mark.parametrize("kwargs,code", BAD_CACHES)
def test_bad_caches_are_refused(call, kwargs, code):
    assert call(cache(**kwargs)) == code
    assert capi.last_error() != ""


@pytest.mark.parametrize("kwargs,code", [
    (dict(dtype=9), capi.FRN_ERR_UNSUPPORTED),
    (dict(Hq=7), capi.FRN_ERR_UNSUPPORTED),
    (dict(Hq=34), capi.FRN_ERR_UNSUPPORTED),
    (dict(batch=-1), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(batch=70000), capi.FRN_ERR_UNSUPPORTED),
    (dict(q=None), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(lens=None), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(q=17), capi.FRN_ERR_MISALIGNED),
    (dict(qs=(1024, 100)), capi.FRN_ERR_MISALIGNED),
    (dict(ws=None), capi.FRN_ERR_WORKSPACE),
    (dict(ws_bytes=100), capi.FRN_ERR_WORKSPACE),
])
def test_paged_decode_refusals(kwargs, code):
    assert decode(cache(), **kwargs) == code
    assert capi.last_error() != ""


@pytest.mark.parametrize("kwargs,code", [
    (dict(dtype=-1), capi.FRN_ERR_UNSUPPORTED),
    (dict(tokens=3), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(tokens=-2), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(k=None), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(start=None), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(k=20), capi.FRN_ERR_MISALIGNED),
    (dict(ks=(256, 4)), capi.FRN_ERR_MISALIGNED),
])
def test_append_refusals(kwargs, code):
    assert append(cache(), **kwargs) == code
    assert capi.last_error() != ""


def test_no_cache_and_nothing_to_do():
    assert decode(None) == append(None) == capi.FRN_ERR_INVALID_ARGUMENT
    assert decode(cache(), batch=0, q=None) == capi.FRN_OK
    assert append(cache(), batch=0, tokens=0, k=None) == capi.FRN_OK


def copy(pools=(16, 32), src=(0,), dst=(1,), num_pages=4, page=64, stride=64):
    import ctypes
    n = len(src)
    return capi.lib().frn_kv_pages_copy(
        (ctypes.c_void_p * max(1, len(pools)))(*pools), len(pools), num_pages, page, stride,
        (ctypes.c_int32 * max(1, n))(*src), (ctypes.c_int32 * max(1, n))(*dst), n, None)


@pytest.mark.parametrize("kwargs,code", [
    (dict(src=(4,)), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(dst=(-1,)), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(src=(0, 1), dst=(2, 2)), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(src=(0, 1), dst=(1, 2)), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(src=(0,), dst=(0,)), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(page=0), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(num_pages=-1), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(page=72, stride=72), capi.FRN_ERR_MISALIGNED),
    (dict(stride=48), capi.FRN_ERR_MISALIGNED),
    (dict(pools=(16, 24)), capi.FRN_ERR_MISALIGNED),
    (dict(pools=(16, None)), capi.FRN_ERR_INVALID_ARGUMENT),
    (dict(page=1 << 30, stride=1 << 30), capi.FRN_ERR_UNSUPPORTED),
])
def test_copy_refusals(kwargs, code):
    assert copy(**kwargs) == code
    assert capi.last_error() != ""


def test_copy_of_nothing():
    assert copy(pools=()) == capi.FRN_OK
    assert copy(src=(), dst=()) == capi.FRN_OK
