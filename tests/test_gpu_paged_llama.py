"""The serving operators together: a tiny patched Llama over the paged cache
against the unpatched model's own forward (packed prompts, decode steps, forks
that diverge, freeing and compaction in mid-flight)."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _models(heads=8, kv_heads=2, hidden=512):
    from transformers import LlamaConfig, LlamaForCausalLM

    from src.paged_llama import PagedLlama
    from src.patch_llama import patch_llama_model

    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=1000, hidden_size=hidden, intermediate_size=1024,
                      num_hidden_layers=2, num_attention_heads=heads,
                      num_key_value_heads=kv_heads, max_position_embeddings=512,
                      rms_norm_eps=1e-5)
    cfg._attn_implementation = "sdpa"
    base = LlamaForCausalLM(cfg).to(torch.bfloat16).to(DEV).eval()
    patched = patch_llama_model(copy.deepcopy(base), variant="V3", swiglu=True)
    return base, PagedLlama(patched, num_pages=40)


def _last_logits(base, tokens):
    with torch.no_grad():
        return base(torch.tensor([tokens], device=DEV)).logits[0, -1]


def _close(got, base, histories):
    for row, tokens in zip(got, histories):
        ref = _last_logits(base, tokens).float()
        rel = ((row.float() - ref).norm() / ref.norm()).item()
        assert rel < 3e-2, f"relative logit error {rel} after {len(tokens)} tokens"


@pytest.mark.parametrize("heads,kv_heads,hidden", [(8, 2, 512), (4, 4, 512)])
def test_serving_matches_the_model(heads, kv_heads, hidden):
    base, server = _models(heads, kv_heads, hidden)
    g = torch.Generator().manual_seed(1)
    texts = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (70, 1, 33)]
    seqs, logits = server.prefill(texts)
    _close(logits, base, texts)
    for step in range(3):
        new = [(7 * step + i) % 1000 for i in range(3)]
        logits = server.decode(seqs, new)
        texts = [t + [n] for t, n in zip(texts, new)]
        _close(logits, base, texts)
    # Forks of the first sequence go different ways; the second one leaves, and
    # the pages are moved together.
    forks = [server.cache.fork(seqs[0]) for _ in range(2)]
    server.cache.free(seqs[1])
    assert server.cache.compact() > 0
    running = [seqs[0], seqs[2]] + forks
    texts = [texts[0], texts[2], list(texts[0]), list(texts[0])]
    for step in range(20):
        new = [(31 * step + 5 * i) % 1000 for i in range(4)]
        logits = server.decode(running, new)
        texts = [t + [n] for t, n in zip(texts, new)]
    _close(logits, base, texts)
    for s in running:
        server.cache.free(s)
    assert server.cache.free_pages == 40


def test_generate_is_greedy():
    base, server = _models()
    prompts = [[5, 9, 300, 4], [17] * 40]
    out = server.generate(prompts, 6)
    assert [len(o) for o in out] == [6, 6] and server.cache.free_pages == 40
    for p, o in zip(prompts, out):
        tokens = list(p)
        for t in o:
            ref = _last_logits(base, tokens).float()
            # Greedy up to near ties: the token is within the logits' error of the best.
            assert ref[t] >= ref.max() - 0.05 * ref.std() * 3
            tokens.append(t)


def test_refusals():
    from src.paged_kv_cache import OutOfPages, PagedKVCache

    _, server = _models()
    with pytest.raises(OutOfPages):
        server.prefill([[1] * 400, [2] * 400])
    assert server.cache.free_pages == 40 and server.cache.sequences() == []
    with pytest.raises(ValueError, match="at least one token"):
        server.prefill([[1], []])
    cache = PagedKVCache(1, 8, 16, 2, 64)
    a = cache.new_sequence()
    cache.extend([a], [3])
    step = cache.extend([a], [2])
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="had tokens"):
        cache.prompt_attention(step, q, q[:, :2], q[:, :2])
    with pytest.raises(ValueError, match="one token"):
        cache.decode_attention(0, step, q)
