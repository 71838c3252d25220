"""Packed and paged sequences and sampling on the CPU: the PyTorch statements against 64-bit loops, their refusals, the paged cache and
``generate(fused_sampling=True)``."""
import pytest
import torch

import oslo_b200 as ob
from oslo_b200 import ops
from oslo_b200.generation import PagedKVCache

from . import plain_serving as plain

REFUSED = (ValueError, RuntimeError)


def rnd(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed + sum(shape))).to(dtype)


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.mark.parametrize("window", [None, 3])
@pytest.mark.parametrize("before", [None, [0, 4, 7, 0]])
def test_ragged_attention_statement(window, before):
    lens = [5, 0, 1, 9]
    klens = [a + b for a, b in zip(lens, before or [0] * 4)]
    q_at, k_at = plain.starts(lens), plain.starts(klens)
    q, k, v, do = (rnd(n, h, 8, seed=i, dtype=torch.bfloat16) for i, (n, h) in enumerate([(17, 4), (k_at[-1] + 2, 2), (k_at[-1] + 2, 2), (17, 4)]))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = ops.ragged_attention(*leaves, ints(*q_at), ints(*k_at) if before else None, window=window)
    want = plain.ragged(q, k, v, q_at, k_at, window, 8 ** -0.5, do)
    plain.near(o.detach(), *want[0])
    assert not o[15:].any()
    for got, (w, b) in zip(torch.autograd.grad(o, leaves, do), want[1:]):
        plain.near(got, w, 2 * b)        # the statement's products are rounded to 16 bits on the way back


def test_ragged_attention_queries_without_keys():
    q, k = rnd(6, 1, 8, seed=1), rnd(2, 1, 8, seed=2)
    o = ops.ragged_attention(q, k, k, ints(0, 6), ints(0, 2))
    assert not o[:4].any() and torch.isfinite(o).all() and o[4:].abs().sum() > 0


@pytest.mark.parametrize("bad", [
    dict(q=(5, 3, 8)), dict(k=(5, 2, 16), v=(5, 2, 16)), dict(v=(4, 2, 8)), dict(offsets=torch.tensor([0, 5])), dict(offsets=ints(5)),
    dict(scale=0.0), dict(window=-1), dict(dtype=torch.float16), dict(key_offsets=ints(0, 2, 5)),
])
def test_ragged_attention_refusals(bad):
    q, k, v = rnd(*bad.get("q", (5, 4, 8))), rnd(*bad.get("k", (5, 2, 8))), rnd(*bad.get("v", (5, 2, 8)))
    with pytest.raises(REFUSED):
        ops.ragged_attention(q.to(bad.get("dtype", q.dtype)), k, v, bad.get("offsets", ints(0, 5)), bad.get("key_offsets"), window=bad.get("window"), scale=bad.get("scale"))


def pool(pages, heads, page, dim, dtype, seed=0):
    k, v = rnd(pages, heads, page, dim, seed=seed), rnd(pages, heads, page, dim, seed=seed + 1)
    if dtype != torch.float8_e4m3fn:
        return k.to(dtype), v.to(dtype), None, None
    (k, ks), (v, vs) = ops.reference.quantise(k), ops.reference.quantise(v)
    return k, v, ks, vs


@pytest.mark.parametrize("store", [torch.float32, torch.float8_e4m3fn])
def test_paged_statements(store):
    kp, vp, ks, vs = pool(9, 2, 4, 16, store)
    table = ints(3, 5, 0, -1, -1, -1, 8, 2, 99).view(3, 3)
    lengths = [10, 0, 7]
    q = rnd(3, 6, 16, seed=5)
    o = ops.paged_attention(q, kp, vp, table, ints(*lengths), k_scale=ks, v_scale=vs)
    for b in (0, 2):
        k, v = plain.held(kp, ks, table, b, lengths[b]), plain.held(vp, vs, table, b, lengths[b])
        for h in range(6):
            p = torch.softmax(k[:, h // 3] @ q[b, h].double() / 4, 0)
            assert torch.allclose(o[b, h].double(), p @ v[:, h // 3], atol=1e-6)
    assert not o[1].any()
    # what is read is what is held; what is appended is what was given, to half a step of e4m3
    k, v = ops.paged_read(kp, vp, table, ints(0, 10, 10, 17), 19, k_scale=ks, v_scale=vs, dtype=torch.float32 if ks is not None else None)
    assert torch.allclose(k[:10].double(), plain.held(kp, ks, table, 0, 10)) and torch.allclose(v[10:17].double(), plain.held(vp, vs, table, 2, 7))
    assert not k[17:].any()
    before = kp.view(torch.uint8).clone() if ks is not None else kp.clone()
    kn, vn = rnd(6, 2, 16, seed=7), rnd(6, 2, 16, seed=8)
    ops.paged_append(kn, vn, kp, vp, table, ints(*lengths), ints(0, 2, 2, 5), k_scale=ks, v_scale=vs)
    step = 2.0 ** -4 if ks is not None else 0
    for b, rows, n in ((0, slice(0, 2), 10), (2, slice(2, 5), 7)):
        got = plain.held(kp, ks, table, b, n)[n - (rows.stop - rows.start):]
        assert ((got - kn[rows].double()).abs() <= step * kn[rows].double().abs() + (2.0 ** -10 * kn[rows].abs().amax(-1, keepdim=True) if step else 0)).all()
    now = kp.view(torch.uint8) if ks is not None else kp
    assert (now != before).flatten(2).any(-1).sum() <= 2 * 6 and (now[1] == before[1]).all()


def test_a_vector_of_zeros_and_one_that_is_no_number():
    x = torch.zeros(4, 16)
    x[1, 3], x[2, 5], x[3, 0] = float("nan"), float("inf"), 1e-30
    y, s = ops.reference.quantise(x)
    back = y.float() * s[:, None]
    assert not back[0].any() and back[1].isnan().all() and back[2].isnan().all() and abs(back[3, 0].item() / 1e-30 - 1) < 2 ** -4


def paged_args(**bad):
    kp, vp, ks, vs = pool(4, 2, 4, 16, bad.pop("store", torch.float32))
    args = dict(q=rnd(2, 4, 16), k_pages=kp, v_pages=vp, page_table=ints(0, 1, 2, 3).view(2, 2), lengths=ints(5, 8), k_scale=ks, v_scale=vs)
    args.update(bad)
    return args


BAD_PAGES = [dict(k_scale=torch.ones(4, 2, 4)), dict(store=torch.float8_e4m3fn, k_scale=None), dict(page_table=torch.zeros(2, 2, dtype=torch.long)),
             dict(v_pages=torch.zeros(4, 2, 4, 8)), dict(store=torch.float8_e4m3fn, v_scale=torch.ones(4, 2, 3)), dict(k_pages=torch.zeros(8, 2, 4, 16)[::2])]


@pytest.mark.parametrize("bad", BAD_PAGES + [dict(q=rnd(3, 4, 16)), dict(q=rnd(2, 3, 16)), dict(lengths=torch.tensor([5, 8])), dict(window=-1),
                                             dict(q=rnd(2, 4, 16, dtype=torch.float16))])
def test_paged_attention_refusals(bad):
    with pytest.raises(REFUSED):
        ops.paged_attention(**paged_args(**bad))


@pytest.mark.parametrize("bad", BAD_PAGES + [dict(k=rnd(3, 2, 16)), dict(v=rnd(2, 1, 16)), dict(offsets=ints(0, 1)), dict(lengths=ints(1)),
                                             dict(k=rnd(2, 2, 16, dtype=torch.float16))])
def test_paged_append_refusals(bad):
    args = paged_args(**{k: v for k, v in bad.items() if k not in ("k", "v", "offsets")})
    args.pop("q")
    with pytest.raises(REFUSED):
        ops.paged_append(bad.get("k", rnd(2, 2, 16)), bad.get("v", rnd(2, 2, 16)), offsets=bad.get("offsets"), **args)


@pytest.mark.parametrize("bad", BAD_PAGES + [dict(offsets=ints(0, 1)), dict(tokens=-1), dict(dtype=torch.float16)])
def test_paged_read_refusals(bad):
    args = paged_args(**{k: v for k, v in bad.items() if k not in ("offsets", "tokens", "dtype")})
    args.pop("q"), args.pop("lengths")
    with pytest.raises(REFUSED):
        ops.paged_read(offsets=bad.get("offsets", ints(0, 1, 2)), tokens=bad.get("tokens", 2), dtype=bad.get("dtype"), **args)


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=3), dict(top_p=0.6), dict(min_p=0.2), dict(temperature=1.3, top_k=20, top_p=0.8, min_p=0.05),
            dict(temperature=0.0), dict(top_k=1), dict(top_p=0.0), dict(min_p=2.0)]


@pytest.mark.parametrize("settings", SETTINGS)
def test_sampling_statement(settings):
    x = 2 * rnd(40, 57, seed=3)
    x[0] = 1.0                                  # equal logits
    x[1, 5:] = float("-inf")
    x[2, 7] = float("nan")
    x[3] = float("-inf")
    x[4, 9] = float("inf")
    x[5, 11] = x[5, 40] = float("inf")
    u = torch.rand(40, generator=torch.Generator().manual_seed(1))
    u[6], u[7] = 0.0, 1.0
    got = ops.sample_tokens(x, u, **settings)
    full = dict(dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **settings)
    assert got.tolist() == plain.sample(x, u, **full).tolist()
    assert got[2] == got[3] == got[7] == -1


def test_sampling_settings_per_row():
    x, u = 2 * rnd(30, 101, seed=4), torch.rand(30, generator=torch.Generator().manual_seed(2))
    g = torch.Generator().manual_seed(3)
    s = dict(temperature=torch.rand(30, generator=g) * 1.5, top_k=torch.randint(0, 8, (30,), generator=g, dtype=torch.int32), top_p=torch.rand(30, generator=g), min_p=0.3 * torch.rand(30, generator=g))
    assert ops.sample_tokens(x, u, **s).tolist() == plain.sample(x, u, **s).tolist()


@pytest.mark.parametrize("bad", [dict(temperature=-1.0), dict(top_k=-1), dict(top_p=-0.1), dict(min_p=-0.1), dict(top_p=float("nan")), dict(uniform=torch.rand(3)),
                                 dict(uniform=torch.zeros(4, dtype=torch.float16)), dict(top_k=torch.ones(4)), dict(temperature=torch.ones(3)), dict(logits=rnd(4))])
def test_sampling_refusals(bad):
    with pytest.raises(REFUSED):
        ops.sample_tokens(**dict(dict(logits=rnd(4, 9), uniform=torch.rand(4)), **bad))


def test_paged_cache_hands_out_and_takes_back_pages():
    cache = PagedKVCache(layers=1, pages=6, page=4, heads=2, dim=16, rows=3, dtype=torch.float32)
    cache.extend([5, 0, 9])
    assert cache.lengths.tolist() == [5, 0, 9] and cache.free_pages == 1
    with pytest.raises(RuntimeError):
        cache.extend([0, 9, 0])
    assert cache.lengths.tolist() == [5, 0, 9] and cache.free_pages == 1
    cache.release(2)
    cache.extend([4, 9, 0])
    assert cache.lengths.tolist() == [9, 9, 0] and cache.free_pages == 0
    used = cache.table[:2, :3].flatten().tolist()
    assert sorted(used) == list(range(6)) and (cache.table[2] == -1).all()


@pytest.mark.parametrize("quantised", [False, True])
def test_prompts_and_steps_through_the_paged_cache(quantised):
    """Prompts of different lengths, one of them going on behind its cached part, then single tokens, against attention over the whole."""
    cache = PagedKVCache(layers=2, pages=20, page=4, heads=2, dim=16, rows=3, dtype=torch.float32, quantised=quantised)
    told = {r: ([], []) for r in range(3)}
    worst = 0.0
    for step, new in enumerate([[6, 1, 0], [3, 0, 11], [1, 1, 1], [1, 1, 1], [1, 0, 1]]):
        n = sum(new)
        q, k, v = (rnd(n, h, 16, seed=10 * step + h + i) for i, h in ((0, 4), (1, 2), (2, 2)))
        cache.extend(new)
        at = plain.starts(new)
        offsets = ints(*at)
        cache.append(1, k, v, offsets)
        if new == [1, 1, 1]:
            o = cache.attend(1, q)
        else:
            kk, vv, key_offsets = cache.read(1)
            o = ops.ragged_attention(q, kk, vv, offsets, key_offsets)
        for r in range(3):
            told[r][0].extend(k[at[r]:at[r + 1]]), told[r][1].extend(v[at[r]:at[r + 1]])
            if new[r]:
                kr, vr = torch.stack(told[r][0]), torch.stack(told[r][1])
                p = plain.softmax(torch.einsum("qhd,khd->hqk", q[at[r]:at[r + 1]].double(), kr.double().repeat_interleave(2, 1)) / 4,
                                  plain.visible(new[r], len(kr), 0, "cpu"))
                want = torch.einsum("hqk,khd->qhd", p, vr.double().repeat_interleave(2, 1))
                worst = max(worst, (o[at[r]:at[r + 1]].double() - want).abs().max().item())
    # e4m3: half a step, 2^-4, of values up to 4 and of scores up to 4 or so
    assert worst < (0.6 if quantised else 1e-5), worst


def tiny():
    cfg = ob.GPT2Config(vocab_size=61, n_positions=64, n_embd=32, n_layer=2, n_head=2)
    torch.manual_seed(0)
    return ob.GPT2LMHeadModel(cfg).eval()


def test_generate_with_fused_sampling():
    model = tiny()
    ids = torch.arange(6).view(2, 3)
    torch.manual_seed(5)
    a = model.generate(ids, do_sample=True, max_length=20, top_k=7, top_p=0.9, temperature=0.8, fused_sampling=True)
    torch.manual_seed(5)
    b = model.generate(ids, do_sample=True, max_length=20, top_k=7, top_p=0.9, temperature=0.8, fused_sampling=True)
    assert a.tolist() == b.tolist() and a.shape == (2, 20)
    # one token kept: what greedy search finds
    greedy = model.generate(ids, max_length=20)
    assert model.generate(ids, do_sample=True, max_length=20, top_k=1, fused_sampling=True).tolist() == greedy.tolist()
    out = model.generate(ids, do_sample=True, max_length=8, top_k=3, fused_sampling=True, min_p=0.1, output_scores=True, return_dict_in_generate=True)
    for i, scores in enumerate(out.scores):      # every token is among the three that the scores keep
        assert torch.isfinite(scores.gather(1, out.sequences[:, 3 + i, None])).all() and (torch.isfinite(scores).sum(1) <= 3).all()


def test_min_p_without_fused_sampling():
    model = tiny()
    ids = torch.arange(6).view(2, 3)
    assert model.generate(ids, do_sample=True, max_length=12, top_k=0, min_p=1.0).tolist() == model.generate(ids, max_length=12).tolist()


def test_min_p_with_beams_is_refused():
    model = tiny()
    with pytest.raises(ValueError, match="one beam"):
        model.generate(torch.tensor([[3, 4]]), num_beams=2, do_sample=True, max_length=6, min_p=0.1)
