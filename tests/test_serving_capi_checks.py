"""The Python wrappers of the serving entry points look at shapes, types and strides before a
pointer goes anywhere: on the CPU, what does not fit is refused."""
import pytest
import torch

from src import capi


def half(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


PROMPT = dict(q=half(9, 4, 64), k=half(9, 2, 64), v=half(9, 2, 64), cu_seqlens=ints(3))
DECODE = dict(q=half(3, 4, 64), k_pages=half(5, 16, 2, 64), v_pages=half(5, 16, 2, 64),
              page_table=ints(3, 2), seq_lens=ints(3))
APPEND = dict(k=half(3, 2, 64), v=half(3, 2, 64), k_pages=half(5, 16, 2, 64),
              v_pages=half(5, 16, 2, 64), page_table=ints(3, 2), start_lens=ints(3))


@pytest.mark.parametrize("change", [
    dict(k=half(8, 2, 64)), dict(v=half(8, 2, 64)), dict(k=half(9, 2, 128)), dict(k=half(9, 1, 64)),
    dict(k=half(9, 2, 64).half()), dict(cu_seqlens=ints(3).long()), dict(cu_seqlens=ints(0)),
    dict(cu_seqlens=ints(3, 2)[:, 0]), dict(v=half(9, 64, 2).transpose(1, 2)),
    dict(out=half(9, 4, 32)), dict(out=half(8, 4, 64)), dict(out=half(9, 4, 64).float())],
    ids=lambda x: "-".join(x))
def test_prompt(change):
    with pytest.raises(AssertionError):
        capi.gqa_prompt_attention(**dict(PROMPT, **change), max_seqlen=9, scale=0.1)


@pytest.mark.parametrize("change", [
    dict(v_pages=half(4, 16, 2, 64)), dict(v_pages=half(5, 8, 2, 64)), dict(page_table=ints(2, 2)),
    dict(seq_lens=ints(2)), dict(seq_lens=ints(3).long()), dict(page_table=ints(3, 2).long()),
    dict(page_table=ints(2, 3).t()), dict(q=half(3, 4, 128)), dict(q=half(3, 4, 64).half()),
    dict(v_pages=half(5, 16, 2, 64).float()), dict(k_pages=half(5, 16, 64, 2).transpose(2, 3)),
    dict(out=half(2, 4, 64)), dict(out=half(3, 4, 64).float())], ids=lambda x: "-".join(x))
def test_decode(change):
    with pytest.raises(AssertionError):
        capi.gqa_paged_decode_attention(**dict(DECODE, **change), scale=0.1)


@pytest.mark.parametrize("change", [
    dict(v=half(2, 2, 64)), dict(k=half(3, 1, 64), v=half(3, 1, 64)), dict(k=half(3, 2, 64).float()),
    dict(start_lens=ints(2)), dict(start_lens=ints(3).long()), dict(page_table=ints(4, 2)),
    dict(cu_seqlens=ints(3)), dict(cu_seqlens=ints(4).long()),
    dict(v=half(3, 64, 2).transpose(1, 2))], ids=lambda x: "-".join(x))
def test_append(change):
    with pytest.raises(AssertionError):
        capi.kv_cache_append(**dict(APPEND, **change))


@pytest.mark.parametrize("pools", [[half(4, 8), half(5, 8)], [half(4, 8), half(4, 8).float()],
                                   [half(4, 8), half(8, 4).t()], [half(8, 4).t()],
                                   [half(4, 2, 16)[:, :, :8]]])
def test_copy(pools):
    with pytest.raises(AssertionError):
        capi.kv_pages_copy(pools, [0], [1])
