"""A tiny patched Llama whose cache is too small for what it is asked to write."""
import pytest
import torch

from src.paged_kv_cache import OutOfPages
from test_gpu_paged_llama import _close, _models

pytestmark = pytest.mark.gpu


def test_generate_out_of_pages():
    base, server = _models()
    with pytest.raises(OutOfPages):
        server.generate([[5] * 300, [7] * 320], 60)  # 19 and 20 of 40 pages, then one each too many
    assert server.cache.free_pages == 40 and server.cache.sequences() == []
    texts = [[5, 9, 300, 4], [17] * 40]
    seqs, logits = server.prefill(texts)
    _close(logits, base, texts)
    for s in seqs:
        server.cache.free(s)
    torch.cuda.synchronize()
