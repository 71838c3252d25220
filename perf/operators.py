"""Operators of a server that keeps its sequences in pages, as a list of measurable cases.

Five kinds of call, each an operator of ``oslo_b200.ops``:

* ``prompt`` / ``train``: ``ragged_attention`` - causal attention with grouped heads over sequences of different lengths that lie one
  behind another; ``train`` returns the gradients too.
* ``append``: ``paged_append`` - new keys and values into the pages of a cache, as they are or quantised to 8 bits.
* ``read``: ``paged_read`` - what the pages hold, one sequence behind another, in 16 bits again.
* ``decode``: ``paged_attention`` - one new token per sequence against its pages.
* ``sample``: ``sample_tokens`` - a token per row of logits with temperature, top-k, top-p and min-p, from given random numbers.

Every input comes from the seed; the lengths come from the case. With ``own`` false ``run`` states the operators in elementary torch
operations; ``exact`` states them in 64 bits, sequence by sequence.
"""
from __future__ import annotations

import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "fp8": torch.float8_e4m3fn}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "fp8": 1}
FP8_MAX = 448.0
LOGIT_SPREAD = 2.5           # standard deviation of a head's logits


# ------------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # a server's step over new prompts: chats of very different lengths behind one another, one of them a single token
        dict(name="prompt_6", kind="prompt", heads=32, kv_heads=8, dim=128, lengths="1531,77,2048,1,640,901", before="", window=0, dtype="bf16"),
        # two long documents at once
        dict(name="prompt_long", kind="prompt", heads=16, kv_heads=4, dim=128, lengths="8192,4099", before="", window=0, dtype="bf16"),
        # fine-tuning on packed conversations, shared key heads
        dict(name="train_7", kind="train", heads=32, kv_heads=8, dim=128, lengths="2048,1500,777,1999,64,311,1493", before="", window=0, dtype="bf16"),
        # GPT-2's heads on packed short texts, 16-bit floats
        dict(name="train_gpt2", kind="train", heads=12, kv_heads=12, dim=64, lengths="1000,1024,333,512,719,65,1001,100,850", before="", window=0,
             dtype="fp16"),
        # a decode step's keys and values, quantised: launch latency
        dict(name="append_64", kind="append", heads=8, dim=128, page=64, rows=64, new=1, longest=4000, mix=1, dtype="bf16", store="fp8"),
        # the prompts of prompt_6 and more, quantised as they are written
        dict(name="append_8000", kind="append", heads=8, dim=128, page=64, rows=8, new=1013, longest=5000, mix=2, dtype="bf16", store="fp8"),
        # a prompt goes on behind a cached part: the part is read back
        dict(name="read_1", kind="read", heads=8, dim=128, page=64, rows=1, longest=1900, mix=3, dtype="bf16", store="fp8"),
        dict(name="read_24", kind="read", heads=8, dim=128, page=64, rows=24, longest=4000, mix=4, dtype="bf16", store="fp8"),
        # one user, and a server's full batch on an 8-bit cache
        dict(name="decode_1", kind="decode", heads=32, kv_heads=8, dim=128, page=64, rows=1, longest=4001, mix=5, window=0, dtype="bf16", store="bf16"),
        dict(name="decode_128", kind="decode", heads=32, kv_heads=8, dim=128, page=64, rows=128, longest=6000, mix=6, window=0, dtype="bf16",
             store="fp8"),
        # one user with the usual settings; a full batch, every row with settings of its own
        dict(name="sample_1", kind="sample", rows=1, vocab=50257, temperature=0.8, top_k=50, top_p=0.95, min_p=0.0, per_row=False, dtype="fp32"),
        dict(name="sample_512", kind="sample", rows=512, vocab=50400, temperature=1.0, top_k=0, top_p=0.9, min_p=0.02, per_row=True, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "train", "train", "append", "read", "decode", "decode", "sample", "sample"])
    dtype = rng.choice(["bf16", "fp16"])
    store = rng.choice(["fp8", dtype])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    if kind in ("prompt", "train"):
        kv_heads, group = rng.choice([1, 2, 4, 8, 12]), rng.choice([1, 2, 3, 4, 4, 6, 8])
        kv_heads = min(kv_heads, 32 // group)
        most = 3 * 10 ** 8 if kind == "train" else 10 ** 9       # padded scores of the plain form
        rows = _log(rng, 1, 24)
        longest = _log(rng, 8, min(8192, int(math.sqrt(most / (rows * kv_heads * group)))))
        lengths = [longest] + [_log(rng, 1, longest) for _ in range(rows - 1)]
        rng.shuffle(lengths)
        before = [0] * rows
        if kind == "prompt" and rng.random() < 0.4:              # continued prompts: cached keys ahead of the new ones
            room = max(1, int(most / (rows * kv_heads * group * longest)) - longest)
            before = [_log(rng, 1, min(4096, room)) - 1 for _ in range(rows)]
        window = _log(rng, 16, 1024) if rng.random() < 0.25 else 0
        return dict(kind=kind, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, lengths=",".join(map(str, lengths)),
                    before=",".join(map(str, before)) if any(before) else "", window=window, dtype=dtype)
    if kind == "sample":
        vocab = _log(rng, 1000, 200000)
        rows = _log(rng, 1, min(512, 20 * 10 ** 6 // vocab))
        return dict(kind=kind, rows=rows, vocab=vocab, temperature=round(rng.uniform(0.3, 1.5), 2), top_k=rng.choice([0, 0, 1, 40, 50, _log(rng, 2, 2000)]),
                    top_p=rng.choice([1.0, 0.8, 0.9, 0.95, round(rng.uniform(0.2, 0.99), 2)]), min_p=rng.choice([0.0, 0.0, 0.05, 0.1]),
                    per_row=rng.random() < 0.5, dtype=rng.choice(["bf16", "fp16", "fp32"]))
    page, rows = rng.choice([16, 32, 64, 64, 128, 48]), _log(rng, 1, 128)
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    longest = min(_log(rng, 16, 16384), 5 * 10 ** 8 // (rows * kv_heads * dim))
    case = dict(kind=kind, dim=dim, page=page, rows=rows, longest=longest, mix=rng.randrange(10 ** 6), dtype=dtype, store=store)
    if kind == "append":
        return dict(case, heads=kv_heads, new=rng.choice([1, 1, min(_log(rng, 2, 2000), max(1, 32000 // rows), longest)]))
    if kind == "read":
        return dict(case, heads=kv_heads, longest=min(longest, 60000 // rows))
    return dict(case, heads=kv_heads * rng.choice([1, 2, 4, 5, 7, 8]), kv_heads=kv_heads, window=_log(rng, 16, 4096) if rng.random() < 0.25 else 0)


def _numbers(text):
    return [int(x) for x in text.split(",")] if text else []


def _cached(case):
    """Tokens that every sequence has in its pages: from few to ``longest``, half of them within a third of it."""
    r = random.Random(case["mix"])
    low = max(1, case.get("new", 1))
    got = [max(low, r.randint(2 * case["longest"] // 3, case["longest"]) if r.random() < 0.5 else r.randint(1, case["longest"])) for _ in range(case["rows"])]
    got[0] = max(low, case["longest"])
    return got


def _starts(lengths):
    got = [0]
    for n in lengths:
        got.append(got[-1] + n)
    return got


# ------------------------------------------------------------------------------------------------------------------ inputs
def _attention_inputs(case, g, dev):
    q_len = _numbers(case["lengths"])
    k_len = [a + b for a, b in zip(q_len, _numbers(case["before"]) or [0] * len(q_len))]
    dtype = TYPES[case["dtype"]]
    shape = lambda n, h: (n, h, case["dim"])  # noqa: E731
    grow = 1.0 + 3.0 * (torch.arange(case["dim"], device=dev) % 37 == 5)          # keys have a few large channels
    make = lambda n, h: torch.randn(shape(n, h), generator=g, device=dev)  # noqa: E731
    q, k, v = make(sum(q_len), case["heads"]), make(sum(k_len), case["kv_heads"]) * grow, make(sum(k_len), case["kv_heads"])
    train = case["kind"] == "train"
    s = dict(q=q.to(dtype).requires_grad_(train), k=k.to(dtype).requires_grad_(train), v=v.to(dtype).requires_grad_(train),
             offsets=torch.tensor(_starts(q_len), dtype=torch.int32, device=dev), longest=max(q_len), longest_k=max(k_len))
    s["key_offsets"] = torch.tensor(_starts(k_len), dtype=torch.int32, device=dev) if case["before"] else None
    if train:
        s["grad"] = make(sum(q_len), case["heads"]).to(dtype)
    return s


def _quantised(x):
    """A vector of 8-bit values and the number that multiplies them, so that the largest becomes 448."""
    x = x.float()
    scale = x.abs().amax(-1) / FP8_MAX
    return (x / torch.where(scale > 0, scale, 1.0)[..., None]).to(torch.float8_e4m3fn), scale


def _cache_inputs(case, g, dev):
    """A pool of pages, more than the sequences need, that they share out in a random order."""
    kv_heads = case.get("kv_heads", case["heads"])
    cached, page, dim = _cached(case), case["page"], case["dim"]
    need = [-(-n // page) for n in cached]
    pages = sum(need) + 7
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((case["rows"], max(need)), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    s = dict(page_table=table, lengths=torch.tensor(cached, dtype=torch.int32, device=dev), k_scale=None, v_scale=None)
    for name in ("k", "v"):
        x = torch.randn(pages, kv_heads, page, dim, generator=g, device=dev, dtype=torch.float16 if case["store"] == "fp8" else TYPES[case["store"]])
        if case["store"] == "fp8":
            x, s[name + "_scale"] = _quantised(x)
        s[name + "_pages"] = x
    return s


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed * 7 + 3)
    if case["kind"] in ("prompt", "train"):
        return dict(_attention_inputs(case, g, dev), case=case)
    if case["kind"] == "sample":
        rows = case["rows"]
        s = dict(case=case, logits=(LOGIT_SPREAD * torch.randn(rows, case["vocab"], generator=g, device=dev)).to(TYPES[case["dtype"]]),
                 uniform=torch.rand(rows, generator=g, device=dev))
        settings = dict(temperature=case["temperature"], top_k=case["top_k"], top_p=case["top_p"], min_p=case["min_p"])
        if case["per_row"]:      # settings of its own for every row, around the case's
            near = lambda v, most: torch.clamp(v * (0.8 + 0.4 * torch.rand(rows, generator=g, device=dev)), max=most)  # noqa: E731
            settings = dict(temperature=near(case["temperature"], 10.0), top_p=near(case["top_p"], 1.0), min_p=near(case["min_p"], 1.0),
                            top_k=near(float(case["top_k"]), float(case["vocab"])).to(torch.int32))
        return dict(s, settings=settings)
    s = dict(_cache_inputs(case, g, dev), case=case)
    dtype = TYPES[case["dtype"]]
    if case["kind"] == "append":
        n = case["rows"] * case["new"]
        s["k"], s["v"] = (torch.randn(n, case["heads"], case["dim"], generator=g, device=dev).to(dtype) for _ in range(2))
        s["offsets"] = torch.arange(case["rows"] + 1, dtype=torch.int32, device=dev) * case["new"] if case["new"] > 1 else None
    elif case["kind"] == "read":
        starts = _starts(_cached(case))
        s["offsets"], s["tokens"] = torch.tensor(starts, dtype=torch.int32, device=dev), starts[-1]
    else:
        s["q"] = torch.randn(case["rows"], case["heads"], case["dim"], generator=g, device=dev).to(dtype)
    return s


# ------------------------------------------------------------------------------------------------------------------ the calls
def run(s):
    return {"prompt": _run_prompt, "train": _run_train, "append": _run_append, "read": _run_read, "decode": _run_decode, "sample": _run_sample}[s["case"]["kind"]](s)


def _run_prompt(s):
    if own:
        from oslo_b200 import ops
        return ops.ragged_attention(s["q"], s["k"], s["v"], s["offsets"], s["key_offsets"], window=s["case"]["window"] or None)
    return _plain_attention(s)


def _run_train(s):
    o = _run_prompt(s)
    return (o.detach(),) + torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["grad"])


def _run_append(s):
    if own:
        from oslo_b200 import ops
        ops.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"], s["lengths"], s["offsets"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    else:
        _plain_append(s)
    return s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]


def _run_read(s):
    if own:
        from oslo_b200 import ops
        return ops.paged_read(s["k_pages"], s["v_pages"], s["page_table"], s["offsets"], s["tokens"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                              dtype=TYPES[s["case"]["dtype"]])
    return _plain_read(s)


def _run_decode(s):
    if own:
        from oslo_b200 import ops
        return ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["lengths"], window=s["case"]["window"] or None,
                                   k_scale=s["k_scale"], v_scale=s["v_scale"])
    return _plain_decode(s)


def _run_sample(s):
    if own:
        from oslo_b200 import ops
        return ops.sample_tokens(s["logits"], s["uniform"], **s["settings"])
    return _plain_sample(s)


# ------------------------------------------------------------------------------------------------------------------ plain forms
def _padded(offsets, longest, rows):
    """Row numbers ``[B, longest]`` of packed sequences (clipped to the last row) and which of them are in the sequence."""
    i = torch.arange(longest, device=offsets.device)
    at = offsets[:-1, None].long() + i
    return at.clamp(max=rows - 1), i < (offsets[1:] - offsets[:-1])[:, None]


def _plain_attention(s):
    case, q, k, v = s["case"], s["q"], s["k"], s["v"]
    ko = s["offsets"] if s["key_offsets"] is None else s["key_offsets"]
    rows, group = q.size(0), case["heads"] // case["kv_heads"]
    qi, q_in = _padded(s["offsets"], s["longest"], rows)
    ki, k_in = _padded(ko, s["longest_k"], k.size(0))
    qp, kp, vp = q.float()[qi], k.float()[ki], v.float()[ki]                                   # [B, S, heads, D]
    qp = qp.transpose(1, 2).unflatten(1, (case["kv_heads"], group))                            # [B, kv, group, Sq, D]
    kp, vp = kp.transpose(1, 2).unsqueeze(2), vp.transpose(1, 2).unsqueeze(2)
    scores = torch.matmul(qp, kp.transpose(-1, -2)) * case["dim"] ** -0.5
    n_q, n_k = (s["offsets"][1:] - s["offsets"][:-1])[:, None, None], (ko[1:] - ko[:-1])[:, None, None]
    at = torch.arange(s["longest"], device=q.device)[None, :, None] + n_k - n_q                # a query's place among the keys
    key = torch.arange(s["longest_k"], device=q.device)[None, None, :]
    seen = (key <= at) & k_in[:, None, :] & q_in[:, :, None]
    if case["window"]:
        seen = seen & (key > at - case["window"])
    seen = seen[:, None, None]
    scores = torch.where(seen, scores, torch.finfo(torch.float32).min)
    p = torch.where(seen, torch.exp(scores - scores.amax(-1, keepdim=True)), 0.0)
    o = torch.matmul(p / p.sum(-1, keepdim=True).clamp(min=1e-30), vp)                         # [B, kv, group, Sq, D]
    row = torch.arange(rows, device=q.device)
    b = torch.searchsorted(s["offsets"].long(), row, right=True) - 1
    return o.flatten(1, 2)[b, :, row - s["offsets"].long()[b]].to(q.dtype)


def _places(s, rows, first, count):
    """For ``count`` tokens of every sequence from position ``first`` on: page and place in it, ``[rows, count]``."""
    at = first[:, None].long() + torch.arange(count, device=first.device)
    page = s["case"]["page"]
    return torch.gather(s["page_table"].long(), 1, at // page), at % page


def _plain_append(s):
    case = s["case"]
    n = case["new"]
    pages, place = _places(s, case["rows"], s["lengths"] - n, n)
    for name in ("k", "v"):
        x = s[name].unflatten(0, (case["rows"], n))                                            # [rows, new, heads, D]
        if s["k_scale"] is not None:
            x, scale = _quantised(x)
            s[name + "_scale"][pages, :, place] = scale
            s[name + "_pages"].view(torch.uint8)[pages, :, place] = x.view(torch.uint8)
        else:
            s[name + "_pages"][pages, :, place] = x.to(s[name + "_pages"].dtype)


def _values(s, name, pages):
    """Whole pages ``[..., heads, page, D]`` in 32 bits."""
    x = s[name + "_pages"]
    if s["k_scale"] is None:
        return x[pages].float()
    return x.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float() * s[name + "_scale"][pages][..., None]


def _plain_read(s):
    row = torch.arange(s["tokens"], device=s["offsets"].device)
    b = torch.searchsorted(s["offsets"].long(), row, right=True) - 1
    at = row - s["offsets"].long()[b]
    page = s["page_table"].long()[b, at // s["case"]["page"]]
    got = []
    for name in ("k", "v"):
        x = s[name + "_pages"]
        if s["k_scale"] is None:
            got.append(x[page, :, at % s["case"]["page"]])
        else:
            x = x.view(torch.uint8)[page, :, at % s["case"]["page"]].view(torch.float8_e4m3fn).float()
            got.append((x * s[name + "_scale"][page, :, at % s["case"]["page"]][..., None]).to(TYPES[s["case"]["dtype"]]))
    return tuple(got)


def _plain_decode(s):
    case = s["case"]
    pages = s["page_table"].clamp(min=0).long()
    k, v = (_values(s, name, pages).transpose(1, 2).flatten(2, 3) for name in ("k", "v"))      # [rows, kv, T, D]
    q = s["q"].float().unflatten(1, (case["kv_heads"], -1))
    scores = torch.matmul(q, k.transpose(-1, -2)) * case["dim"] ** -0.5
    at = torch.arange(k.size(2), device=q.device)
    seen = at < s["lengths"][:, None]
    if case["window"]:
        seen = seen & (at >= s["lengths"][:, None] - case["window"])
    scores = torch.where(seen[:, None, None], scores, torch.finfo(torch.float32).min)
    p = torch.where(seen[:, None, None], torch.exp(scores - scores.amax(-1, keepdim=True)), 0.0)
    return torch.matmul(p / p.sum(-1, keepdim=True).clamp(min=1e-30), v).flatten(1, 2).to(s["q"].dtype)


def _plain_sample(s):
    """In 64 bits: a token is chosen by comparing sums with a given number."""
    x, vocab = s["logits"].double(), s["case"]["vocab"]
    get = lambda name: torch.as_tensor(s["settings"][name], dtype=torch.float64, device=x.device).reshape(-1, 1)  # noqa: E731
    w = torch.exp((x - x.amax(1, keepdim=True)) / get("temperature"))
    order = torch.sort(s["logits"], dim=1, descending=True, stable=True).indices               # equal ones: the lowest index first
    rank = torch.arange(vocab, device=x.device)[None]
    top_k = get("top_k")
    ranked = torch.gather(w, 1, order) * ((top_k <= 0) | (rank < top_k))
    before = torch.cumsum(ranked, 1) - ranked
    keep = (ranked > 0) & (ranked >= get("min_p")) & ((get("top_p") >= 1) | (before <= get("top_p") * ranked.sum(1, keepdim=True)) | (rank == 0))
    mass = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ranked, 0.0))
    sums = torch.cumsum(mass, 1)
    return (sums <= s["uniform"].double()[:, None] * sums[:, -1:]).sum(1)


# ------------------------------------------------------------------------------------------------------------------ bytes and operations
def _pairs(case):
    total = 0
    q_len = _numbers(case["lengths"])
    for n, before in zip(q_len, _numbers(case["before"]) or [0] * len(q_len)):
        w = case["window"] or before + n
        total += sum(min(w, before + i + 1) for i in range(n))
    return total


def work(case):
    kind = case["kind"]
    if kind in ("prompt", "train"):
        q_len = _numbers(case["lengths"])
        rows, keys = sum(q_len), sum(q_len) + sum(_numbers(case["before"]))
        size, d = SIZE[case["dtype"]], case["dim"]
        once = 2 * rows * case["heads"] * d + 2 * keys * case["kv_heads"] * d                  # q, o, k, v
        products = _pairs(case) * case["heads"] * d * 2
        if kind == "prompt":
            return {"bytes": once * size, "flops": 2 * products}
        return {"bytes": (2 * once + rows * case["heads"] * d) * size, "flops": 7 * products}    # gradients as large, and the output's
    if kind == "sample":
        return {"bytes": case["rows"] * case["vocab"] * SIZE[case["dtype"]], "flops": 4 * case["rows"] * case["vocab"]}
    cached = _cached(case)
    vector = lambda store: case["dim"] * SIZE[store] + (4 if store == "fp8" else 0)  # noqa: E731
    if kind == "append":
        n = 2 * case["rows"] * case["new"] * case["heads"]
        return {"bytes": n * (vector(case["dtype"]) + vector(case["store"])), "flops": 3 * n * case["dim"]}
    if kind == "read":
        n = 2 * sum(cached) * case["heads"]
        return {"bytes": n * (vector(case["dtype"]) + vector(case["store"])), "flops": n * case["dim"]}
    seen = sum(min(n, case["window"] or n) for n in cached)
    return {"bytes": 2 * seen * case["kv_heads"] * vector(case["store"]) + 2 * case["rows"] * case["heads"] * vector(case["dtype"]),
            "flops": 4 * seen * case["heads"] * case["dim"]}


# ------------------------------------------------------------------------------------------------------------------ in 64 bits
def _exact_attention(case, s):
    group, scale = case["heads"] // case["kv_heads"], case["dim"] ** -0.5
    q_at = _starts(_numbers(case["lengths"]))
    k_at = s["key_offsets"].tolist() if s["key_offsets"] is not None else q_at
    q, k, v = (s[n].detach() for n in ("q", "k", "v"))
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    dq, dk, dv = torch.zeros_like(o), torch.zeros(k.shape, dtype=torch.float64, device=q.device), torch.zeros(v.shape, dtype=torch.float64, device=q.device)
    for b in range(len(q_at) - 1):
        qs, ks = slice(q_at[b], q_at[b + 1]), slice(k_at[b], k_at[b + 1])
        n, m = qs.stop - qs.start, ks.stop - ks.start
        ahead = torch.arange(m, device=q.device)[None] - (torch.arange(n, device=q.device)[:, None] + m - n)
        hidden = ahead > 0
        if case["window"]:
            hidden |= ahead <= -case["window"]
        for h in range(case["heads"]):
            qh, kh, vh = q[qs, h].double(), k[ks, h // group].double(), v[ks, h // group].double()
            p = torch.softmax((qh @ kh.T * scale).masked_fill_(hidden, -math.inf), -1)
            o[qs, h] = p @ vh
            if case["kind"] == "train":
                do = s["grad"][qs, h].double()
                ds = do @ vh.T
                ds -= (ds * p).sum(-1, keepdim=True)
                ds *= p
                dv[ks, h // group] += p.T @ do
                dq[qs, h] = ds @ kh * scale
                dk[ks, h // group] += ds.T @ qh * scale
    return (o, dq, dk, dv) if case["kind"] == "train" else o


def exact(case, seed):
    if case["kind"] == "sample":
        return None
    s = prepare(case, seed)
    if case["kind"] in ("prompt", "train"):
        return _exact_attention(case, s)
    cached, page = _cached(case), case["page"]

    def row(b, name):                                                                          # [tokens, heads, D]
        pages = s["page_table"][b, :-(-cached[b] // page)].long()
        x = s[name + "_pages"].view(torch.uint8)[pages].view(torch.float8_e4m3fn).double() * s[name + "_scale"][pages].double()[..., None] \
            if s["k_scale"] is not None else s[name + "_pages"][pages].double()
        return x.transpose(1, 2).flatten(0, 1)[:cached[b]]

    if case["kind"] == "read":
        return tuple(torch.cat([row(b, name) for b in range(case["rows"])]) for name in ("k", "v"))
    if case["kind"] == "append":
        out = {n: None if s[n] is None else s[n].double() for n in ("k_pages", "v_pages", "k_scale", "v_scale")}
        for b in range(case["rows"]):
            at = torch.arange(cached[b] - case["new"], cached[b], device=s["lengths"].device)
            pages, place = s["page_table"][b].long()[at // page], at % page
            for name in ("k", "v"):
                x = s[name][b * case["new"]:(b + 1) * case["new"]].double()
                if s["k_scale"] is not None:
                    scale = x.abs().amax(-1) / FP8_MAX
                    out[name + "_scale"][pages, :, place] = scale
                    x = x / scale[..., None]
                out[name + "_pages"][pages, :, place] = x
        return out["k_pages"], out["v_pages"], out["k_scale"], out["v_scale"]
    out = torch.empty(case["rows"], case["heads"], case["dim"], dtype=torch.float64, device=s["q"].device)
    for b in range(case["rows"]):
        k, v = (row(b, name)[-case["window"] if case["window"] else 0:].transpose(0, 1) for name in ("k", "v"))
        q = s["q"][b].double().unflatten(0, (case["kv_heads"], -1))
        out[b] = (torch.softmax(q @ k.transpose(1, 2) * case["dim"] ** -0.5, -1) @ v).flatten(0, 1)
    return out
