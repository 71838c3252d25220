"""The kernels of packed and paged sequences and of sampling against 64-bit loops (``plain_serving.py``, which derives the bounds)."""
import pytest
import torch

import oslo_b200 as ob
from oslo_b200 import ops
from oslo_b200.generation import PagedKVCache

from . import plain_serving as plain

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
FP8 = torch.float8_e4m3fn


def rnd(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed + 7919 * len(shape) + sum(shape))
    return (scale * torch.randn(*shape, generator=g)).to(dtype).cuda()


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------------------------------ packed attention
def ragged_case(heads, kv, dim, lens, before=None, window=None, dtype=BF16, lead=0, tail=0, seed=0, grads=True):
    klens = [a + b for a, b in zip(lens, before or [0] * len(lens))]
    q_at, k_at = [x + lead for x in plain.starts(lens)], [x + lead for x in plain.starts(klens)]
    q, do = (rnd(q_at[-1] + tail, heads, dim, seed=seed + i, dtype=dtype) for i in (1, 2))
    k, v = (rnd(k_at[-1] + tail, kv, dim, seed=seed + i, dtype=dtype) for i in (3, 4))
    leaves = [t.clone().requires_grad_(grads) for t in (q, k, v)]
    o = ops.ragged_attention(*leaves, ints(*q_at), ints(*k_at) if before or lead else None, window=window)
    want = plain.ragged(q, k, v, q_at, k_at, window, dim ** -0.5, do if grads else None)
    plain.near(o.detach(), *(want[0] if grads else want))
    if grads:
        for got, (w, b) in zip(torch.autograd.grad(o, leaves, do), want[1:]):
            plain.near(got, w, b)


@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 64), (8, 2, 128), (4, 1, 256), (6, 2, 80), (7, 1, 96), (16, 1, 64), (10, 5, 8), (12, 4, 192), (64, 1, 16)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_ragged_heads(heads, kv, dim, dtype):
    ragged_case(heads, kv, dim, [1, 129, 0, 64, 257, 3], dtype=dtype)


@pytest.mark.parametrize("lens", [[1], [127], [128], [129], [513], [1, 1, 1, 1, 1], [0, 0, 5], [300, 0, 0], [64, 64, 64], [31, 33, 400, 2, 255, 256, 257]])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 128), (3, 3, 64), (2, 1, 256)])
def test_ragged_lengths(lens, heads, kv, dim):
    ragged_case(heads, kv, dim, lens, seed=7)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window", [1, 2, 100, 128, 1000])
def test_ragged_windows(dim, window):
    ragged_case(4, 2, dim, [300, 1, 700], window=window, seed=9)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window", [None, 70])
def test_ragged_keys_ahead_of_the_queries(dim, window):
    ragged_case(4, 1, dim, [1, 130, 5, 64], [500, 3, 0, 129], window=window, seed=11)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_ragged_fewer_keys_than_queries(dim):
    """The first queries see nothing: zeros, and no gradient passes through them."""
    ragged_case(4, 2, dim, [200, 300, 64, 9], [-150, -300, -1, -8], seed=13)


@pytest.mark.parametrize("heads,kv", [(4, 4), (4, 1)])
def test_ragged_rows_of_no_sequence(heads, kv):
    ragged_case(heads, kv, 64, [130, 7], lead=37, tail=200, seed=15)
    ragged_case(heads, kv, 128, [130, 7], lead=300, tail=1, seed=16)


def test_ragged_many_sequences():
    ragged_case(8, 2, 64, [1 + (i * 37) % 61 for i in range(150)], seed=17)


def test_ragged_far_scores():
    """Scores of hundreds: weights of nearly one and nearly nothing."""
    q, k, v = (rnd(500, 2, 64, seed=i, dtype=BF16, scale=s) for i, s in ((1, 12.0), (2, 4.0), (3, 1.0)))
    o = ops.ragged_attention(q, k, v, ints(0, 200, 500))
    w, b = plain.ragged(q, k, v, [0, 200, 500], [0, 200, 500], None, 0.125)
    # scores up to 1200 in 32 bits: the exponent is off by up to 1200 * 2^-23 or so
    near = b + 2.0 ** -12 * v.double().abs().amax()
    plain.near(o, w, near)


def test_ragged_strided_and_joint_projections():
    """Slices of one projection: the gradients are slices of one tensor."""
    x = rnd(300, (4 + 2 + 2) * 64, seed=3, dtype=BF16).requires_grad_()
    q, k, v = (x[:, a:b].view(300, -1, 64) for a, b in ((0, 256), (256, 384), (384, 512)))
    at = [0, 100, 300]
    o = ops.ragged_attention(q, k, v, ints(*at))
    do = rnd(4, 300, 64, seed=4, dtype=BF16).transpose(0, 1)                   # an odd order
    want = plain.ragged(q.detach(), k.detach(), v.detach(), at, at, None, 0.125, do)
    plain.near(o.detach(), *want[0])
    (dx,) = torch.autograd.grad(o, x, do)
    for part, (w, b) in zip((dx[:, :256], dx[:, 256:384], dx[:, 384:]), want[1:]):
        plain.near(part.reshape(w.shape), w, b)
    # a transposed operand and one that starts between 16-byte boundaries
    qt = q.detach().transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.empty(300 * 2 * 64 + 3, dtype=BF16, device="cuda")[3:].view(300, 2, 64).copy_(k.detach())
    assert torch.equal(ops.ragged_attention(qt, odd, v.detach(), ints(*at)), o.detach())


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_ragged_sequences_do_not_touch_each_other(dim, what):
    """What is no number in one sequence, or in rows of none, leaves the others as they are - forward and backward."""
    at = [0, 100, 170, 330]
    q, k, v, do = (rnd(340, h, dim, seed=i, dtype=BF16) for i, h in enumerate((4, 2, 2, 4)))
    clean = [t.clone().requires_grad_() for t in (q, k, v)]
    o1 = ops.ragged_attention(*clean, ints(*at))
    g1 = torch.autograd.grad(o1, clean, do)
    for t in (q, k, v, do):
        t[100:170] = what
        t[330:] = what
    bad = [t.clone().requires_grad_() for t in (q, k, v)]
    o2 = ops.ragged_attention(*bad, ints(*at))
    g2 = torch.autograd.grad(o2, bad, do)
    for a, b in zip((o1, *g1), (o2, *g2)):
        assert torch.equal(a[:100], b[:100]) and torch.equal(a[170:330], b[170:330])
        assert not b[330:].any()


def test_ragged_gradients_against_differences():
    q, k, v, do = (rnd(40, h, 16, seed=i, dtype=FP16) for i, h in enumerate((4, 2, 2, 4)))
    at = [0, 13, 40]
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.ragged_attention(*leaves, ints(*at)), leaves, do)
    for i in range(3):
        d = rnd(*leaves[i].shape, seed=20 + i, dtype=torch.float64)
        step = 2.0 ** -10

        def loss(sign):
            x = [t.double() for t in (q, k, v)]
            x[i] = x[i] + sign * step * d
            total = 0.0
            for b in range(2):
                s = slice(at[b], at[b + 1])
                n = at[b + 1] - at[b]
                seen = plain.visible(n, n, None, "cuda")
                for h in range(4):
                    p = plain.softmax(x[0][s, h] @ x[1][s, h // 2].T / 4, seen)
                    total += ((p @ x[2][s, h // 2]) * do[s, h].double()).sum().item()
            return total

        want = (loss(1) - loss(-1)) / (2 * step)
        _, *bounds = plain.ragged(q, k, v, at, at, None, 0.25, do)
        room = (bounds[i][1] * d.abs()).sum().item() + 4 * step ** 2 * d.abs().sum().item()
        assert abs((grads[i].double() * d).sum().item() - want) <= room


def test_ragged_captured_and_replayed_with_other_lengths():
    q, k, v = (rnd(256, h, 128, seed=i, dtype=BF16) for i, h in enumerate((4, 2, 2)))
    at = ints(0, 100, 256)
    ops.ragged_attention(q, k, v, at)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = ops.ragged_attention(q, k, v, at)
    for cut in (100, 1, 0, 255):
        at.copy_(ints(0, cut, 256))
        g.replay()
        assert torch.equal(o, ops.ragged_attention(q, k, v, ints(0, cut, 256)))


def test_ragged_is_the_same_every_time_and_on_another_stream():
    q, k, v, do = (rnd(700, h, 128, seed=i, dtype=BF16) for i, h in enumerate((8, 2, 2, 8)))
    at = ints(0, 130, 131, 700)

    def both():
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        o = ops.ragged_attention(*leaves, at)
        return (o.detach(), *torch.autograd.grad(o, leaves, do))

    first = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(first, other, both()):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_ragged_without_rows_and_without_keys():
    q, k = rnd(0, 4, 64, dtype=BF16), rnd(5, 2, 64, dtype=BF16)
    assert ops.ragged_attention(q, k, k, ints(0, 0), ints(0, 5)).shape == (0, 4, 64)
    leaves = [rnd(5, 4, 64, dtype=BF16).requires_grad_(), rnd(0, 2, 64, dtype=BF16).requires_grad_(), rnd(0, 2, 64, dtype=BF16).requires_grad_()]
    o = ops.ragged_attention(*leaves, ints(0, 5), ints(0, 0))
    assert not o.any()
    assert not torch.autograd.grad(o.sum(), leaves[0])[0].any()


def test_ragged_second_derivatives_are_refused():
    leaves = [rnd(5, 2, 64, seed=i, dtype=BF16).requires_grad_() for i in range(3)]
    (g,) = torch.autograd.grad(ops.ragged_attention(*leaves, ints(0, 5)).float().pow(2).sum(), leaves[0], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().sum(), leaves[1])


@pytest.mark.parametrize("window", [131, 2 ** 31 - 1])
def test_ragged_windows_wider_than_all_keys(window):
    # more queries than keys: the first ones stand ahead of every key, and a window reaches far beyond those
    ragged_case(4, 2, 64, [260, 9], [-200, 62], window=window, seed=77)


@pytest.mark.parametrize("bad", [dict(offsets=torch.tensor([0, 5])), dict(offsets=torch.tensor([0, 5]), move=True), dict(scale=-1.0), dict(window=-1), dict(heads=3),
                                 dict(key_offsets=(0, 2, 5)), dict(offsets=torch.tensor([0, 5], dtype=torch.int32))])
def test_ragged_refusals(bad):
    q, k = rnd(5, bad.get("heads", 4), 64, dtype=BF16), rnd(5, 2, 64, dtype=BF16)
    offsets = bad.get("offsets", ints(0, 5))
    offsets = offsets.cuda() if bad.get("move") else offsets
    with pytest.raises((ValueError, RuntimeError)):
        ops.ragged_attention(q, k, k, offsets, ints(*bad["key_offsets"]) if "key_offsets" in bad else None, window=bad.get("window"), scale=bad.get("scale"))


# ------------------------------------------------------------------------------------------------------------------ pages
def paged(lengths, kv, dim, page, store, dtype=BF16, spare=3, seed=0):
    """Pools with more pages than needed, a table in random order, unused entries -1, and garbage in unused rows."""
    need = [-(-n // page) for n in lengths]
    pages, columns = sum(need) + spare, max(need + [1]) + 1
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lengths), columns), -1, dtype=torch.int32)
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(need):
        for i in range(n):
            table[b, i] = order.pop()
            used[table[b, i], :max(0, min(page, lengths[b] - i * page))] = True
    out = [table.cuda(), ints(*lengths)]
    for i in range(2):
        x = rnd(pages, kv, page, dim, seed=seed + i, dtype=dtype)
        if store == FP8:
            x, s = ops.reference.quantise(x * (1 + 30 * torch.rand(pages, kv, page, 1, device="cuda")))
            s.masked_fill_(~used.cuda()[:, None], float("nan"))
        else:
            x.masked_fill_(~used.cuda()[:, None, :, None], float("nan"))
            s = None
        out.append((x, s))
    return out


@pytest.mark.parametrize("store", [BF16, FP16, FP8])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (4, 4, 64), (4, 1, 256), (16, 1, 128), (5, 1, 80), (34, 2, 64), (6, 6, 16), (8, 4, 192)])
def test_paged_attention_heads(heads, kv, dim, store):
    dtype = BF16 if store == FP8 else store
    for q_type in ((BF16, FP16) if store == FP8 else (dtype,)):
        lengths = [1, 700, 0, 64, 65]
        table, lens, (kp, ks), (vp, vs) = paged(lengths, kv, dim, 64, store, dtype, seed=heads)
        q = rnd(5, heads, dim, seed=3, dtype=q_type)
        o = ops.paged_attention(q, kp, vp, table, lens, k_scale=ks, v_scale=vs)
        plain.near(o, *plain.decode(q, kp, vp, table, lengths, None, dim ** -0.5, ks, vs))
        assert not o[2].any()


@pytest.mark.parametrize("page", [1, 7, 16, 48, 100, 256])
@pytest.mark.parametrize("store", [BF16, FP8])
def test_paged_attention_page_sizes(page, store):
    lengths = [333, 1, page, page + 1, 2 * page - 1]
    table, lens, (kp, ks), (vp, vs) = paged(lengths, 2, 64, page, store, seed=page)
    q = rnd(5, 6, 64, seed=page, dtype=BF16)
    o = ops.paged_attention(q, kp, vp, table, lens, k_scale=ks, v_scale=vs)
    plain.near(o, *plain.decode(q, kp, vp, table, lengths, None, 0.125, ks, vs))


@pytest.mark.parametrize("window", [1, 33, 64, 5000])
@pytest.mark.parametrize("rows", [1, 9])
def test_paged_attention_windows_and_long_rows(window, rows):
    lengths = [4097, 3, 100, 0, 64, 1000, 31, 32, 33][:rows]
    table, lens, (kp, _), (vp, _) = paged(lengths, 1, 128, 32, BF16, seed=5)
    q = rnd(rows, 8, 128, seed=6, dtype=BF16)
    plain.near(ops.paged_attention(q, kp, vp, table, lens, window=window), *plain.decode(q, kp, vp, table, lengths, window, 128 ** -0.5))


def test_paged_attention_many_rows_and_strided_queries():
    lengths = [(i * 53) % 300 for i in range(200)]
    table, lens, (kp, ks), (vp, vs) = paged(lengths, 4, 64, 16, FP8, seed=8)
    q = rnd(200, 3, 8 * 64, seed=9, dtype=BF16)[:, 1].view(200, 8, 64)          # rows of a joint projection
    plain.near(ops.paged_attention(q, kp, vp, table, lens, k_scale=ks, v_scale=vs), *plain.decode(q, kp, vp, table, lengths, None, 0.125, ks, vs))


def test_paged_attention_behind_two_gigabytes():
    """Pages whose addresses need more than 32 bits."""
    pages = 2 ** 31 // (2 * 32 * 256) + 40          # elements of a pool: more than 2^31
    kp = torch.zeros(pages * 2, 2, 32, 128, dtype=FP16, device="cuda")
    vp = torch.zeros_like(kp)
    last = ints(pages * 2 - 1, 3, pages + 7).view(1, 3)
    for p in last[0].tolist():
        kp[p], vp[p] = rnd(2, 32, 128, seed=p % 97, dtype=FP16), rnd(2, 32, 128, seed=p % 89, dtype=FP16)
    q = rnd(1, 4, 128, seed=2, dtype=FP16)
    plain.near(ops.paged_attention(q, kp, vp, last, ints(80)), *plain.decode(q, kp, vp, last, [80], None, 128 ** -0.5))
    k, v = rnd(1, 2, 128, seed=3, dtype=FP16), rnd(1, 2, 128, seed=4, dtype=FP16)
    ops.paged_append(k, v, kp, vp, ints(pages * 2 - 1).view(1, 1), ints(32))
    assert torch.equal(kp[-1, :, 31], k[0]) and torch.equal(vp[-1, :, 31], v[0])
    got, _ = ops.paged_read(kp, vp, last, ints(0, 33), 33)
    assert torch.equal(got[31], k[0])


def test_paged_numbers_outside_their_range_are_passed_over():
    """Page numbers, positions and lengths that do not exist: nothing is followed, nothing else changes."""
    table, lens, (kp, _), (vp, _) = paged([64, 64], 2, 64, 16, BF16, seed=3)
    bad = table.clone()
    bad[0, 1], bad[0, 2] = 10 ** 6, -5
    q = rnd(2, 4, 64, seed=1, dtype=BF16)
    got = ops.paged_attention(q, kp, vp, bad, lens)
    at = torch.cat([torch.arange(16), torch.arange(48, 64)]).cuda()
    k, v = plain.held(kp, None, table, 0, 64)[at], plain.held(vp, None, table, 0, 64)[at]
    p = torch.softmax(torch.einsum("hd,khd->hk", q[0].double(), k.repeat_interleave(2, 1)) / 8, 1)
    assert (got[0].double() - torch.einsum("hk,khd->hd", p, v.repeat_interleave(2, 1))).abs().max() < 0.05
    full = ops.paged_attention(q, kp, vp, table, lens)
    assert torch.equal(got[1], full[1])
    assert torch.equal(ops.paged_attention(q, kp, vp, table[:, :4].contiguous(), ints(10 ** 9, 64)), full)      # clamped to the table
    assert not ops.paged_attention(q, kp, vp, table, ints(-3, 64))[0].any()
    was = kp.clone().nan_to_num(7.0), vp.clone().nan_to_num(7.0)
    new = rnd(4, 2, 64, seed=5, dtype=BF16)
    ops.paged_append(new, new, kp, vp, bad, ints(34, 0), ints(0, 2, 3))           # positions 32, 33 (page -5); no length; a row of none
    ops.paged_append(new, new, kp, vp, bad, ints(10 ** 6, -1), ints(0, 2, 4))
    assert torch.equal(kp.nan_to_num(7.0), was[0]) and torch.equal(vp.nan_to_num(7.0), was[1])
    k, _ = ops.paged_read(kp, vp, bad, ints(3, 40, 41), 50)
    assert not k[:3].any() and not k[19:40].any() and not k[41:].any() and torch.equal(k[3:19].double(), plain.held(kp, None, table, 0, 16))


@pytest.mark.parametrize("store", [BF16, FP16, FP8])
@pytest.mark.parametrize("kv,dim,page", [(2, 128, 64), (1, 64, 16), (5, 256, 7), (3, 80, 33), (8, 16, 64)])
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [0, 300, 17, 1], None])
def test_paged_append_and_read(store, kv, dim, page, new):
    dtype = BF16 if store == FP8 else store
    lengths = [5, 700, 64, 130]
    table, lens, (kp, ks), (vp, vs) = paged(lengths, kv, dim, page, store, dtype, seed=dim + page)
    n = 4 if new is None else sum(new)
    both = rnd(n + 2, 2 * kv * dim, seed=4, dtype=dtype, scale=3.0)
    k, v = (both[:, i * kv * dim:(i + 1) * kv * dim].view(-1, kv, dim)[:n if new is None else n + 2] for i in (0, 1))
    if store == FP8:
        k[0, 0] = 0
    # the statement on copies of the pools must have the same bits
    copies = [t.clone() if t is not None else None for t in (kp, vp, ks, vs)]
    off = None if new is None else ints(*plain.starts(new))
    ops.paged_append(k, v, kp, vp, table, lens, off, k_scale=ks, v_scale=vs)
    ops.reference.paged_append(k, v, copies[0], copies[1], table, lens, off, copies[2], copies[3])
    bits = lambda t: t.view(torch.uint8) if t.dtype == FP8 else t.view(torch.int16) if t.element_size() == 2 else t.view(torch.int32)  # noqa: E731
    for got, want in zip((kp, vp, ks, vs), copies):
        if got is not None:
            assert torch.equal(bits(got), bits(want))
    at = plain.starts(lengths)
    rk, rv = ops.paged_read(kp, vp, table, ints(*at), at[-1] + 3, k_scale=ks, v_scale=vs, dtype=dtype)
    for b, m in enumerate(lengths):
        for r, p, s in ((rk, kp, ks), (rv, vp, vs)):
            want = plain.held(p, s, table, b, m)
            assert ((r[at[b]:at[b + 1]].double() - want).abs() <= plain.U[dtype] * want.abs() * (s is not None) + 2.0 ** -24 * (s is not None)).all()
    assert not rk[at[-1]:].any() and not rv[at[-1]:].any()


def test_paged_append_no_numbers_in_8_bits():
    kp, vp = (torch.zeros(2, 1, 8, 32, dtype=torch.uint8, device="cuda").view(FP8) for _ in range(2))
    ks, vs = (torch.zeros(2, 1, 8, device="cuda") for _ in range(2))
    x = rnd(4, 1, 32, dtype=BF16)
    x[0, 0, 3], x[1, 0, 31], x[2] = float("nan"), float("-inf"), 0.0
    ops.paged_append(x, x, kp, vp, ints(1).view(1, 1), ints(4), ints(0, 4), k_scale=ks, v_scale=vs)
    k, v = ops.paged_read(kp, vp, ints(1).view(1, 1), ints(0, 4), 4, k_scale=ks, v_scale=vs, dtype=BF16)
    assert k[0].isnan().all() and k[1].isnan().all() and not k[2].any() and torch.isfinite(k[3]).all()


@pytest.mark.parametrize("bad", [dict(page_table=torch.zeros(2, 2, dtype=torch.long)), dict(lengths=torch.tensor([1, 2])), dict(q=(3, 4, 64)), dict(q=(2, 3, 64)), dict(window=-1),
                                 dict(lengths=torch.ones(2, dtype=torch.int32), cpu=True), dict(store=FP8, drop=True), dict(type=FP16)])
def test_paged_refusals(bad):
    table, lens, (kp, ks), (vp, vs) = paged([5, 9], 2, 64, 8, bad.get("store", BF16))
    if "page_table" in bad:
        table = bad["page_table"].cuda()
    if "lengths" in bad:
        lens = bad["lengths"] if bad.get("cpu") else bad["lengths"].cuda()
    q = rnd(*bad.get("q", (2, 4, 64)), dtype=bad.get("type", BF16))
    with pytest.raises((ValueError, RuntimeError)):
        ops.paged_attention(q, kp, vp, table, lens, window=bad.get("window"), k_scale=None if bad.get("drop") else ks, v_scale=vs)
    if "q" not in bad and "window" not in bad:
        k = rnd(2, 2, 64, dtype=bad.get("type", BF16))
        with pytest.raises((ValueError, RuntimeError)):
            ops.paged_append(k, k, kp, vp, table, lens, k_scale=None if bad.get("drop") else ks, v_scale=vs)


# ------------------------------------------------------------------------------------------------------------------ sampling
SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=3), dict(top_p=0.6), dict(min_p=0.05), dict(temperature=1.3, top_k=200, top_p=0.8, min_p=0.01), dict(top_p=0.999),
            dict(temperature=0.0), dict(top_k=1), dict(top_p=0.0), dict(min_p=2.0), dict(temperature=0.01), dict(temperature=50.0, top_p=0.5), dict(top_k=900, top_p=0.99)]


@pytest.mark.parametrize("settings", SETTINGS)
@pytest.mark.parametrize("rows,vocab,dtype", [(1, 50257, torch.float32), (3, 1000, BF16), (70, 257, FP16), (300, 1, torch.float32), (40, 5003, torch.float32), (2, 131072, BF16)])
def test_sampling(settings, rows, vocab, dtype):
    x, u = rnd(rows, vocab, seed=vocab, dtype=dtype, scale=2.5), torch.rand(rows, generator=torch.Generator().manual_seed(rows)).cuda()
    full = dict(dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **settings)
    assert torch.equal(ops.sample_tokens(x, u, **settings), ops.reference.sample_tokens(x, u, **full))


@pytest.mark.parametrize("settings", SETTINGS)
@pytest.mark.parametrize("vocab", [7, 3001, 30011])
def test_sampling_equal_logits(settings, vocab):
    """Rows of one value, of two, of few: what is kept is decided by the index."""
    x = rnd(24, vocab, seed=1)
    x[:6] = 0.25
    x[6:12] = (x[6:12] > 0).float()
    x[12:18] = x[12:18].round()
    x[18, 1:] = float("-inf")
    x[19] = -0.0
    x[19, ::2] = 0.0
    u = torch.rand(24, generator=torch.Generator().manual_seed(vocab)).cuda()
    u[0], u[1] = 0.0, 1 - 2.0 ** -24
    full = dict(dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **settings)
    assert torch.equal(ops.sample_tokens(x, u, **settings), ops.reference.sample_tokens(x, u, **full))


def test_sampling_against_a_loop():
    x, u = rnd(50, 301, seed=5, scale=2.0), torch.rand(50, dtype=torch.float64, generator=torch.Generator().manual_seed(2)).cuda()
    g = torch.Generator().manual_seed(3)
    s = dict(temperature=torch.rand(50, generator=g) * 1.5, top_k=torch.randint(0, 40, (50,), generator=g, dtype=torch.int32), top_p=torch.rand(50, generator=g), min_p=0.3 * torch.rand(50, generator=g))
    s = {k: v.cuda() for k, v in s.items()}
    s["temperature"][3] = 0.0
    assert ops.sample_tokens(x, u, **s).tolist() == plain.sample(x, u, **s).tolist()


def test_sampling_rows_without_a_choice():
    x, u = rnd(8, 4099, seed=6), torch.full((8,), 0.5, device="cuda")
    x[0, 4000], x[1], x[2, 17], x[3, 17], x[3, 4098] = float("nan"), float("-inf"), float("inf"), float("inf"), float("inf")
    u[4], u[5], u[6] = 1.0, -0.1, float("nan")
    for s in (dict(), dict(top_k=50, top_p=0.9), dict(temperature=0.0), dict(min_p=0.1)):
        got = ops.sample_tokens(x, u, **s)
        assert got[0] == got[1] == got[4] == got[5] == got[6] == -1 and got[2] == 17 and got[7] >= 0
        assert got[3] == (17 if "temperature" in s else 4098 if not s or "min_p" in s or "top_k" in s else 17)


@pytest.mark.parametrize("vocab,dtype", [(400000, torch.float32), (800000, BF16), (400001, torch.float32)])
def test_sampling_the_widest_rows(vocab, dtype):
    x, u = rnd(3, vocab, seed=7, dtype=dtype), torch.tensor([0.0, 0.4, 0.999], device="cuda")
    for s in (dict(), dict(top_k=64, top_p=0.9), dict(top_p=0.95)):
        full = dict(dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **s)
        assert torch.equal(ops.sample_tokens(x, u, **s), ops.reference.sample_tokens(x, u, **full))


def test_sampling_strides_and_alignment():
    wide = rnd(9, 5010, seed=8, dtype=BF16)
    u = torch.rand(9, generator=torch.Generator().manual_seed(1)).cuda()
    for x in (wide[:, 3:5000], wide[:, 1:2], wide[::2, 7:], wide.t().contiguous().t()):
        for s in (dict(top_p=0.9), dict(top_k=9)):
            full = dict(dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **s)
            assert torch.equal(ops.sample_tokens(x, u[:x.size(0)].contiguous(), **s), ops.reference.sample_tokens(x, u[:x.size(0)], **full))


def test_sampling_follows_the_probabilities():
    x = rnd(1, 64, seed=9, scale=1.5)
    u = torch.rand(200000, generator=torch.Generator().manual_seed(4)).cuda()
    got = ops.sample_tokens(x.expand(200000, 64), u, temperature=0.9, top_k=20)
    kept = torch.topk(x[0], 20).indices
    p = torch.zeros(64, device="cuda").scatter(0, kept, torch.softmax(x[0, kept] / 0.9, 0))
    share = torch.bincount(got, minlength=64) / 200000
    assert (share - p).abs().max() < 5 * (0.25 / 200000) ** 0.5          # five standard deviations at most


@pytest.mark.parametrize("bad", [dict(top_k=torch.ones(4)), dict(temperature=torch.ones(3)), dict(uniform=torch.rand(3)), dict(uniform=torch.zeros(4, dtype=FP16)), dict(top_p=-1.0),
                                 dict(logits=torch.zeros(4, 9, dtype=torch.int64))])
def test_sampling_refusals(bad):
    args = dict(dict(logits=torch.zeros(4, 9), uniform=torch.rand(4)), **bad)
    with pytest.raises((ValueError, RuntimeError)):
        ops.sample_tokens(**{k: v.cuda() if torch.is_tensor(v) else v for k, v in args.items()})


# ------------------------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("quantised", [False, True])
def test_a_server_from_prompts_to_tokens(quantised):
    """Prompts of different lengths, one that goes on behind its cached part, and captured single steps, each ending in a token, against
    the same over whole tensors in 64 bits."""
    rows, heads, kv, dim, vocab = 3, 8, 2, 64, 997
    cache = PagedKVCache(layers=1, pages=40, page=16, heads=kv, dim=dim, rows=rows, device="cuda", quantised=quantised)
    head = rnd(heads * dim, vocab, seed=99, scale=0.1)
    told = [([], []) for _ in range(rows)]

    def tell(k, v, at):
        for r in range(rows):
            told[r][0].append(k[at[r]:at[r + 1]].clone())       # the step's buffers are written again
            told[r][1].append(v[at[r]:at[r + 1]].clone())

    def check(o, q, at):
        """Against what the cache holds, and (8 bits) what it holds against what was given: half a step of e4m3."""
        for r in range(rows):
            n = at[r + 1] - at[r]
            if not n:
                continue
            for given, pool, scale in zip(told[r], (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
                have, want = plain.held(pool[0], scale[0], cache.table, r, cache.lengths[r].item()), torch.cat(given).double()
                assert have.shape == want.shape and ((have - want).abs() <= (2.0 ** -4 * want.abs() + 2.0 ** -9 * want.abs().amax(-1, keepdim=True) if quantised else 0)).all()
            k, v = (plain.held(pool[0], scale[0], cache.table, r, cache.lengths[r].item()).to(BF16) for pool, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
            w, b = plain.ragged(q[at[r]:at[r + 1]], k, v, [0, n], [0, k.size(0)], None, dim ** -0.5)
            plain.near(o[at[r]:at[r + 1]], w, b + (2.0 ** -6 * v.double().abs().amax() if quantised else 0))     # read back in 16 bits or not: 2^-8 of scores and values

    for step, new in enumerate([[40, 1, 0], [13, 0, 77], [1, 2, 1]]):
        n, at = sum(new), plain.starts(new)
        q, k, v = (rnd(n, h, dim, seed=10 * step + i, dtype=BF16) for i, h in enumerate((heads, kv, kv)))
        cache.extend(new)
        cache.append(0, k, v, ints(*at))
        kk, vv, key_offsets = cache.read(0)
        o = ops.ragged_attention(q, kk, vv, ints(*at), key_offsets)
        tell(k, v, at)
        check(o, q, at)
    # single tokens: one captured step, replayed on new inputs and a table that changes on the host
    q, k, v, u = rnd(rows, heads, dim, seed=70, dtype=BF16), rnd(rows, kv, dim, seed=71, dtype=BF16), rnd(rows, kv, dim, seed=72, dtype=BF16), torch.zeros(rows, device="cuda")

    def one():
        cache.append(0, k, v)
        o = cache.attend(0, q)
        logits = o.flatten(1).float() @ head
        return o, logits, ops.sample_tokens(logits, u, temperature=0.8, top_k=50, top_p=0.9)

    cache.extend([1, 1, 1])
    one()
    torch.cuda.synchronize()
    tell(k, v, [0, 1, 2, 3])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o, logits, tokens = one()
    for step in range(20):
        cache.extend([1, 1, 1])
        for t, s in ((q, 100), (k, 200), (v, 300)):
            t.copy_(rnd(*t.shape, seed=s + step, dtype=BF16))
        u.copy_(torch.rand(rows, generator=torch.Generator().manual_seed(step)))
        g.replay()
        tell(k, v, [0, 1, 2, 3])
        check(o, q, [0, 1, 2, 3])
        assert torch.equal(tokens, ops.reference.sample_tokens(logits, u, 0.8, 50, 0.9, 0.0))
    cache.release(1)
    assert cache.attend(0, q)[1].abs().max() == 0


def test_generate_with_fused_sampling_on_the_gpu():
    torch.manual_seed(0)
    model = ob.GPT2LMHeadModel(ob.GPT2Config(vocab_size=50257, n_positions=64, n_embd=128, n_layer=2, n_head=2)).cuda().to(BF16).eval().fuse()
    ids = torch.arange(6, device="cuda").view(2, 3)
    greedy = model.generate(ids, max_length=20)
    assert torch.equal(model.generate(ids, do_sample=True, max_length=20, top_k=1, fused_sampling=True), greedy)
    out = model.generate(ids, do_sample=True, max_length=30, top_k=5, top_p=0.9, fused_sampling=True, output_scores=True, return_dict_in_generate=True)
    for i, scores in enumerate(out.scores):
        assert torch.isfinite(scores.gather(1, out.sequences[:, 3 + i, None])).all()
