"""Cases for measuring the serving attention operators: attention over packed prompts, decode
attention over a paged key-value cache, appending tokens to the pages, and copying pages.

``own`` chooses between the plain form of each operator (elementary torch operations in 32 bits,
rounded once) and the calls a user makes of this framework.  Head layouts are those of the models
the framework patches: 32 query / 8 key-value heads of 128 (the Llama QKV sweep), 64 heads with
192-wide keys and 128-wide values (what q_b and kv_b produce for the MLA layers), and the smaller
layouts of the decode-attention tests.
"""
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
LAYERS = 32  # layers whose K and V pools one page move covers


def _gqa():
    """The framework's attention entry points."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    project = os.path.join(root, "kimi26-h100-rmsnorm-swiglu-fusion_b200")
    if project not in sys.path:
        sys.path.insert(0, project)
    from src.load_gqa_attention import gqa_attention_cuda
    return gqa_attention_cuda


def listed():
    return [
        # One short chat turn on a small GQA model: what counts is latency.
        _prompt("prompt_short", 1, 77, 77, 28, 4, 64, 64, "fp16"),
        # A prefill batch of a server: requests of very different lengths, packed.
        _prompt("prompt_packed", 24, 16, 1500, 32, 8, 128, 128, "bf16"),
        # One long document.
        _prompt("prompt_long", 1, 8192, 8192, 32, 8, 128, 128, "bf16"),
        # A prefill batch of the MLA layers, V a strided view of kv_b's output.
        _prompt("prompt_mla", 4, 500, 2048, 64, 64, 192, 128, "bf16"),
        # One user, one stream: latency of a single token.
        _decode("decode_one", 1, 1000, 1000, 32, 8, 128, 16, "bf16"),
        # A continuous batch in mid-flight, an idle slot in it.
        _decode("decode_batch", 64, 1, 8192, 32, 8, 128, 16, "bf16"),
        # A few very long contexts.
        _decode("decode_long", 8, 100000, 131072, 32, 8, 128, 64, "bf16"),
        # 32-bit evaluation of a small model.
        _decode("decode_fp32", 3, 500, 2000, 16, 2, 64, 32, "fp32"),
        # The new tokens of one decode step.
        _append("append_step", 64, 1, 1, 8, 128, 16, "bf16"),
        # The keys and values of freshly prefilled prompts.
        _append("append_prompts", 16, 200, 4000, 8, 128, 64, "fp16"),
        # Copy-on-write of the last page when eight sequences are forked, all layers.
        _copy("copy_fork", 8, 64, 2 * LAYERS, 16, 8, 128, "bf16"),
        # Compaction of a fragmented cache, all layers.
        _copy("copy_compact", 1001, 2600, 2 * LAYERS, 16, 8, 128, "bf16"),
    ]


def draw(rng):
    def log(low, high):
        return int(round(low * (high / low) ** rng.random()))

    op = rng.choice(["prompt", "prompt", "decode", "decode", "append", "copy"])
    if op == "prompt":
        batch = log(1, 32)
        longest = log(16, int(8192 / batch ** 0.5))
        hq, hkv, d, dv = rng.choice([(32, 8, 128, 128), (28, 4, 64, 64), (16, 2, 64, 64),
                                     (8, 8, 128, 128), (12, 4, 128, 128), (64, 64, 192, 128)])
        if d == 192:
            longest = max(16, longest // 2)
        return _prompt(None, batch, log(1, longest), longest, hq, hkv, d, dv,
                       rng.choice(["bf16", "fp16"]), rng.randrange(1 << 30))
    hq, hkv, d = rng.choice([(32, 8, 128), (28, 4, 128), (16, 2, 64), (8, 8, 64), (32, 2, 128)])
    page = rng.choice([8, 16, 24, 32, 64, 128])
    if op == "decode":
        batch = log(1, 256)
        longest = log(16, min(131072, 1000000 // batch))
        return _decode(None, batch, log(1, longest), longest, hq, hkv, d, page,
                       rng.choice(["bf16", "fp16", "bf16", "fp16", "fp32"]), rng.randrange(1 << 30))
    if op == "append":
        batch = log(1, 256)
        longest = log(1, max(1, 65536 // batch))
        return _append(None, batch, log(1, longest), longest, hkv, d, page,
                       rng.choice(["bf16", "fp16", "fp32"]), rng.randrange(1 << 30))
    return _copy(None, log(1, 800), 1700, 2 * log(1, LAYERS), rng.choice([8, 16, 24]), hkv, d,
                 rng.choice(["bf16", "fp16"]), rng.randrange(1 << 30))


def _named(case, name):
    return case if name is None else dict(case, name=name)


def _prompt(name, batch, low, high, hq, hkv, d, dv, dtype, mix=1):
    return _named(dict(op="prompt", batch=batch, low=low, high=high, hq=hq, hkv=hkv, d=d, dv=dv,
                       dtype=dtype, mix=mix), name)


def _decode(name, batch, low, high, hq, hkv, d, page, dtype, mix=2):
    return _named(dict(op="decode", batch=batch, low=low, high=high, hq=hq, hkv=hkv, d=d, dv=d,
                       page=page, dtype=dtype, mix=mix), name)


def _append(name, batch, low, high, hkv, d, page, dtype, mix=3):
    return _named(dict(op="append", batch=batch, low=low, high=high, hkv=hkv, d=d, page=page,
                       dtype=dtype, mix=mix), name)


def _copy(name, pairs, pages, pools, page, hkv, d, dtype, mix=4):
    return _named(dict(op="copy", pairs=pairs, pages=pages, pools=pools, page=page, hkv=hkv, d=d,
                       dtype=dtype, mix=mix), name)


def _lens(case):
    """Sequence lengths: spread over the logarithm between `low` and `high`, both ends among them;
    a decode batch of more than eight has one empty slot."""
    rng = random.Random(case["mix"])
    low, high, n = case["low"], case["high"], case["batch"]
    lens = [int(round(low * (high / low) ** rng.random())) for _ in range(n)]
    lens[-1] = high
    if n > 1:
        lens[0] = low
    rng.shuffle(lens)
    if case["op"] == "decode" and n > 8 and lens[n // 2] != high:
        lens[n // 2] = 0
    return lens


def _ceil(a, b):
    return -(-a // b)


def work(case):
    es = BYTES[case["dtype"]]
    if case["op"] == "copy":
        page = case["page"] * case["hkv"] * case["d"] * es
        return {"bytes": 2 * case["pairs"] * case["pools"] * page, "flops": 0}
    lens = _lens(case)
    total = sum(lens)
    if case["op"] == "append":
        return {"bytes": 4 * total * case["hkv"] * case["d"] * es, "flops": 0}
    hq, hkv, d, dv = (case[k] for k in ("hq", "hkv", "d", "dv"))
    if case["op"] == "decode":
        return {"bytes": total * hkv * (d + dv) * es + case["batch"] * hq * (d + dv) * es
                + 4 * sum(_ceil(n, case["page"]) for n in lens) + 4 * case["batch"],
                "flops": 2 * total * hq * (d + dv)}
    return {"bytes": total * (hq + hkv) * (d + dv) * es + 4 * (case["batch"] + 1),
            "flops": sum(n * (n + 1) for n in lens) * hq * (d + dv)}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", dtype=dt, generator=g)

    if case["op"] == "copy":
        pools = [normal(case["pages"], case["page"], case["hkv"], case["d"])
                 for _ in range(case["pools"])]
        order = random.Random(seed).sample(range(case["pages"]), 2 * case["pairs"])
        return dict(op="copy", pools=pools, src=order[:case["pairs"]], dst=order[case["pairs"]:])
    lens = _lens(case)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)

    def ints(values):
        return torch.tensor(values, device="cuda", dtype=torch.int32)

    if case["op"] == "prompt":
        q = normal(cu[-1], case["hq"], case["d"])
        if case["d"] == case["dv"]:
            k, v = (normal(cu[-1], case["hkv"], case["d"]) for _ in range(2))
        else:  # V is the tail of each head's [nope | V] block
            k = normal(cu[-1], case["hkv"], case["d"])
            v = normal(cu[-1], case["hkv"], 128 + case["dv"])[..., 128:]
        return dict(op="prompt", q=q, k=k, v=v, cu=ints(cu), longest=max(lens),
                    scale=case["d"] ** -0.5)
    # A cache that has been in use: pages of a sequence lie anywhere, unused entries are -1.
    page = case["page"]
    before = [0] * len(lens)
    if case["op"] == "append":
        rng = random.Random(case["mix"] + 1)
        before = [rng.randrange(0, 200) for _ in lens]
    need = [_ceil(n + m, page) for n, m in zip(lens, before)]
    spare = 3
    order = random.Random(seed).sample(range(sum(need) + spare), sum(need))
    width = max(need) + 1
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    k_pages, v_pages = (normal(sum(need) + spare, page, case["hkv"], case["d"]) for _ in range(2))
    state = dict(op=case["op"], k_pages=k_pages, v_pages=v_pages, table=ints(table))
    if case["op"] == "decode":
        return dict(state, q=normal(len(lens), case["hq"], case["d"]), lens=ints(lens),
                    scale=case["d"] ** -0.5)
    k, v = (normal(cu[-1], case["hkv"], case["d"]) for _ in range(2))
    return dict(state, k=k, v=v, before=ints(before), cu=None if max(lens) == 1 else ints(cu))


def run(state):
    if own:
        ops = _gqa()
        if state["op"] == "prompt":
            return ops.gqa_prompt_attention(state["q"], state["k"], state["v"], state["cu"],
                                            state["longest"], state["scale"])
        if state["op"] == "decode":
            return ops.gqa_paged_decode(state["q"], state["k_pages"], state["v_pages"],
                                        state["table"], state["lens"], state["scale"])
        if state["op"] == "append":
            ops.kv_cache_append(state["k"], state["v"], state["k_pages"], state["v_pages"],
                                state["table"], state["before"], state["cu"])
            return state["k_pages"], state["v_pages"]
        ops.kv_pages_copy(state["pools"], state["src"], state["dst"])
        return state["pools"]
    return {"prompt": _plain_prompt, "decode": _plain_decode, "append": _plain_append,
            "copy": _plain_copy}[state["op"]](state)


def _softmax_times(scores, keep, v, product):
    """softmax(scores where keep) times v; a row with nothing to keep gives zeros."""
    scores = scores.masked_fill_(~keep, float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)
    scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    scores.div_(total.clamp_(min=torch.finfo(torch.float32).tiny))
    return torch.einsum(product, scores, v)


def _plain_prompt(s):
    """Sequences padded to the longest, all scores at once, a causal mask."""
    q, k, v, cu, longest = s["q"], s["k"], s["v"], s["cu"].long(), s["longest"]
    lens = cu[1:] - cu[:-1]
    at = torch.arange(longest, device=q.device)
    there = at[None] < lens[:, None]
    rows = (cu[:-1, None] + at[None]).clamp(max=q.size(0) - 1)
    hkv = k.size(1)
    qp = q[rows].float().unflatten(2, (hkv, q.size(1) // hkv))
    scores = torch.einsum("bihgd,bjhd->bhgij", qp, k[rows].float()).mul_(s["scale"])
    out = _softmax_times(scores, at[:, None] >= at[None], v[rows].float(), "bhgij,bjhd->bihgd")
    return out.flatten(2, 3)[there].to(q.dtype)


def _plain_decode(s):
    """Every sequence's pages gathered into one padded cache."""
    q, table, lens = s["q"], s["table"].long().clamp(min=0), s["lens"].long()
    k, v = (s[n][table].flatten(1, 2).float() for n in ("k_pages", "v_pages"))
    hkv = k.size(2)
    qg = q.float().unflatten(1, (hkv, q.size(1) // hkv))
    scores = torch.einsum("bhgd,bthd->bhgt", qg, k).mul_(s["scale"])
    keep = torch.arange(k.size(1), device=q.device)[None] < lens[:, None]
    out = _softmax_times(scores, keep[:, None, None], v, "bhgt,bthd->bhgd")
    return out.flatten(1, 2).to(q.dtype)


def _plain_append(s):
    k, before, page = s["k"], s["before"].long(), s["k_pages"].size(1)
    token = torch.arange(k.size(0), device=k.device)
    cu = token if s["cu"] is None else s["cu"].long()[:-1]
    seq = torch.searchsorted(cu, token, right=True) - 1
    position = before[seq] + token - cu[seq]
    pages = s["table"].long()[seq, position // page]
    s["k_pages"][pages, position % page] = k
    s["v_pages"][pages, position % page] = s["v"]
    return s["k_pages"], s["v_pages"]


def _plain_copy(s):
    src, dst = (torch.tensor(s[n], device="cuda") for n in ("src", "dst"))
    for pool in s["pools"]:
        pool[dst] = pool[src]
    return s["pools"]


def exact(case, seed):
    if case["op"] not in ("prompt", "decode"):
        return None  # copies: no arithmetic
    s = prepare(case, seed)
    q = s["q"]
    out = torch.zeros(*q.shape[:2], case["dv"], dtype=torch.float64, device=q.device)
    group = case["hq"] // case["hkv"]
    first = 0
    for b, n in enumerate(_lens(case)):
        if case["op"] == "prompt":
            mine = slice(first, first + n)
            k, v = s["k"][mine], s["v"][mine]
            first += n
        else:
            mine = slice(b, b + 1)
            pages = s["table"][b, :_ceil(n, case["page"])].long()
            k, v = (s[x][pages].reshape(-1, case["hkv"], case["d"])[:n]
                    for x in ("k_pages", "v_pages"))
        if n == 0:
            continue
        for h in range(case["hq"]):
            kh, vh = k[:, h // group].double(), v[:, h // group].double()
            a = (q[mine, h].double() @ kh.T) * s["scale"]
            if case["op"] == "prompt":
                a += torch.full_like(a, float("-inf")).triu_(1)
            a = torch.exp(a - a.max(dim=1, keepdim=True).values)
            out[mine, h] = (a @ vh) / a.sum(dim=1, keepdim=True)
    return out
