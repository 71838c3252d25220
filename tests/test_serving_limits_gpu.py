"""Serving operators where their inputs are at a limit: infinities and what is no number, rows of a cluster, borders of a sum, 16-bit
ranges. The statements in 64 bits and their bounds are ``plain_serving``'s."""
import pytest
import torch

from oslo_b200 import ops
from oslo_b200.ops.cuda_ops import _op

from . import plain_serving as plain

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def rnd(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed + 7919 * len(shape) + sum(shape))
    return (scale * torch.randn(*shape, generator=g)).to(dtype).cuda()


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def settings_of(**given):
    return dict(dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **given)


# ------------------------------------------------------------------------------------------------------------------ sampling
@pytest.mark.parametrize("vocab,dtype", [(50257, BF16), (50257, torch.float32), (50001, FP16)])
@pytest.mark.parametrize("others", [1.0, 8.0])
def test_sampling_counts_a_token_once_where_blocks_meet(vocab, dtype, others):
    """Rows that several blocks share, whose starts lie between 16-byte boundaries, with the largest logits around every place where one
    block's tokens may end and another's begin (a quarter and an eighth of the row, rounded up to 16)."""
    places = sorted({(-(-vocab // c) + 15) // 16 * 16 * i + d for c in (2, 4, 8) for i in range(1, c) for d in range(-8, 9)})
    places = [at for at in places if at < vocab]
    for shift in range(8):          # every start of a row with every place
        for first in range(0, len(places), 24):
            some = places[first:first + 24]
            some = some[shift:] + some[:shift]
            x = rnd(len(some), vocab, seed=first + shift).to(dtype)
            rows = torch.arange(len(some), device="cuda")
            x[rows, torch.tensor(some, device="cuda")] = 30.0
            x[rows, torch.tensor([at - 1 for at in some], device="cuda")] = 30.0 - others      # 1: both are kept; 8: one
            for u in (0.1, 0.45, 0.55, 0.99):
                uniform = torch.full((len(some),), u, device="cuda")
                got = ops.sample_tokens(x, uniform, top_p=0.9)
                assert torch.equal(got, ops.reference.sample_tokens(x, uniform, **settings_of(top_p=0.9))), (shift, first, u)


@pytest.mark.parametrize("rows,vocab,dtype", [(1, 50257, torch.float32), (40, 50257, BF16), (300, 5003, torch.float32), (160, 30011, FP16), (6, 131072, torch.float32)])
@pytest.mark.parametrize("temperature,spread", [(1.0, 2.5), (0.7, 1.0)])
def test_sampling_at_the_border_of_top_p(rows, vocab, dtype, temperature, spread):
    """Top-p within half a step of 32 bits (2^-25) of the share at which a token is kept or not. That token has the largest index, so the
    largest ``uniform`` chooses it if it is kept. What is nearer than 2^-30 is left out: weights are good to 4e-11, some 2^-34."""
    x = rnd(rows, vocab, seed=rows, scale=spread).to(dtype)
    last = vocab - 1
    r = torch.arange(rows, device="cuda")
    share = torch.tensor([0.3, 0.5, 0.9, 0.97, 0.999], device="cuda", dtype=torch.float64)[r % 5]

    def ahead_of_each(x):
        order = torch.sort(x.double(), dim=1, descending=True, stable=True).indices
        w = torch.exp((x.double() - x.double().amax(1, keepdim=True)) / temperature)
        ranked = torch.gather(w, 1, order)
        return order, torch.cumsum(ranked, 1) - ranked, w.sum(1, keepdim=True)

    order, ahead, whole = ahead_of_each(x)
    rank = (ahead < share[:, None] * whole).sum(1).clamp(max=last)          # the first token behind that share
    token = torch.gather(order, 1, rank[:, None])[:, 0]
    swapped = x[r, token].clone()
    x[r, token] = x[:, last].clone()
    x[:, last] = swapped
    order, ahead, whole = ahead_of_each(x)
    at = (order == last).nonzero()[:, 1]
    border = ahead[r, at] / whole[:, 0]
    top_p = border.float()
    told = (top_p.double() - border).abs() > 2.0 ** -30
    uniform = torch.full((rows,), 1 - 2.0 ** -24, device="cuda")
    s = settings_of(temperature=temperature, top_p=top_p)
    want = ops.reference.sample_tokens(x, uniform, **s)
    assert torch.equal((want == last)[told], (border <= top_p.double())[told])
    got = ops.sample_tokens(x, uniform, temperature=temperature, top_p=top_p)
    assert torch.equal(got[told], want[told])
    s["min_p"] = 1e-7          # the same border
    assert torch.equal(ops.sample_tokens(x, uniform, **s)[told], ops.reference.sample_tokens(x, uniform, **s)[told])


@pytest.mark.parametrize("given", [dict(), dict(top_k=3), dict(top_k=700), dict(top_p=0.6), dict(top_k=700, top_p=0.6), dict(min_p=0.5), dict(temperature=0.0)])
@pytest.mark.parametrize("dtype", [torch.float32, BF16, FP16])
@pytest.mark.parametrize("vocab", [9, 5003, 50257])
def test_sampling_rows_of_the_lowest_values(given, dtype, vocab):
    """Logits at and near the type's lowest value, which masks write, and minus infinity."""
    low = torch.finfo(dtype).min
    x = torch.full((8, vocab), low, dtype=dtype, device="cuda")
    x[1, 1::3] = float("-inf")
    x[2, 5:] = float("-inf")
    x[3, ::2] = low * (1 - 2.0 ** -6)
    x[4] = low * (1 - 0.03125 * torch.rand(vocab, generator=torch.Generator().manual_seed(1))).to(dtype).cuda()
    x[5, 7] = 0.0
    x[6, ::5] = -1.0
    x[7, 2] = low / 2
    u = torch.tensor([0.5, 0.9, 0.3, 0.7, 0.2, 0.6, 0.99, 0.1], device="cuda")
    assert torch.equal(ops.sample_tokens(x, u, **given), ops.reference.sample_tokens(x, u, **settings_of(**given)))


@pytest.mark.parametrize("given", [dict(), dict(top_k=3), dict(top_k=700), dict(top_p=0.6), dict(top_k=700, top_p=0.6), dict(min_p=0.5)])
@pytest.mark.parametrize("dtype", [torch.float32, BF16, FP16])
@pytest.mark.parametrize("temperature", [1e-36, 1e-6, 1e-3, 1.0, 1e4])
def test_sampling_logits_far_larger_than_the_temperature(given, dtype, temperature):
    """Logits around a value at which 32-bit steps are wider than the temperature, or not so much."""
    vocab, rows = 5003, 10
    most = torch.finfo(dtype).max * (1 - 2.0 ** -6)
    at = torch.tensor([3e38, -3e38, 1e30, -1e20, 1e12, 6e4, -6e4, 1e3, -30.0, 1.0]).clamp(-most, most)
    x = (at[:, None] * (1 + 2.0 ** -9 * torch.randint(-3, 4, (rows, vocab), generator=torch.Generator().manual_seed(2)))).to(dtype).cuda()
    x[:, 7::11] = float("-inf")
    u = torch.tensor([0.5, 0.9, 0.3, 0.7, 0.2, 0.6, 0.99, 0.1, 0.0, 0.45], device="cuda")
    assert x.isfinite().any(1).all() and not x.isnan().any() and not (x == float("inf")).any()
    # weights are whole multiples of 2^-45 of the largest: what rounds to none is not chosen, not even by a uniform number of 0
    weighs = torch.exp((x.double() - x.double().amax(1, keepdim=True)) / temperature) >= 2.0 ** -46
    want = ops.reference.sample_tokens(x.masked_fill(~weighs, float("-inf")), u, **settings_of(temperature=temperature, **given))
    assert torch.equal(ops.sample_tokens(x, u, temperature=temperature, **given), want)


def test_sampling_settings_that_are_no_numbers():
    """Per row: the first of the largest logits, on a GPU as on the CPU."""
    x, u = rnd(12, 3001, seed=3), torch.full((12,), 0.9, device="cuda")
    x[:, 5] = x[:, 77] = 9.0
    nan = torch.full((12,), float("nan"), device="cuda")
    for given in (dict(temperature=nan), dict(top_p=nan), dict(min_p=nan), dict(top_p=nan, top_k=900), dict(min_p=nan, top_k=40)):
        full = settings_of(**given)
        assert (ops.sample_tokens(x, u, **given) == 5).all()
        assert (ops.reference.sample_tokens(x.cpu(), u.cpu(), **{k: v.cpu() if torch.is_tensor(v) else v for k, v in full.items()}) == 5).all()


# ------------------------------------------------------------------------------------------------------------------ packed attention
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
def test_ragged_a_key_that_is_no_number(dim, dtype, what):
    """Sequence i has one bad value in key i. With NaN rows ahead of it are as they were, bit by bit, and all others are NaN. With an infinity
    rows whose score becomes plus infinity, or that see no other key, are NaN, and the others as if that key were not there - to the bound
    of a result of its own, not to the bit: a row's weights are rounded relative to a reference that may follow those of its neighbours,
    and an infinite score makes that follow."""
    count, length = 70, 83
    at = plain.starts([length] * count)
    q, k, v = (rnd(count * length, h, dim, seed=i, dtype=dtype) for i, h in enumerate((2, 1, 1)))
    clean = ops.ragged_attention(q, k, v, ints(*at))
    bad = k.clone()
    for i in range(count):
        bad[at[i] + i, 0, 3] = what
    got = ops.ragged_attention(q, bad, v, ints(*at))
    seen = plain.visible(length, length, None, "cuda")
    u = plain.U[dtype]
    for i in range(count):
        a, mid, z = at[i], at[i] + i, at[i + 1]
        if what != what:
            assert torch.equal(got[a:mid], clean[a:mid]) and got[mid:z].isnan().all()
            continue
        assert q[a:z, :, 3].ne(0).all()
        up = (q[a:z, :, 3].float() * what > 0) & (torch.arange(length, device="cuda") >= i)[:, None]
        if i == 0:
            up[0] = True                                # sees nothing else
        assert torch.equal(got[a:z].isnan().all(-1), up) and torch.equal(got[a:z].isnan().any(-1), up)
        keep = [j for j in range(length) if j != i]
        vv = v[a:z, 0].double()[keep]
        for h in range(2):
            p = plain.softmax((q[a:z, h].double() @ k[a:z, 0].double().T * dim ** -0.5)[:, keep], seen[:, keep])
            w = p @ vv
            over = (got[a:z, h].double() - w).abs() - ((u + plain.SMALL) * (p @ vv.abs()) + u * w.abs() + 2.0 ** -24)
            assert over[~up[:, h]].max() <= 0


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("window", [None, 2])
def test_ragged_a_query_that_is_no_number(dim, dtype, window):
    """One bad query in each sequence, at its first places too, where a row meets few keys: its row is NaN and no other."""
    lens = [1] + [20] * 20 + [70, 130]
    at = plain.starts(lens)
    where = [0] + list(range(20)) + [66, 129]
    q, k, v = (rnd(at[-1], h, dim, seed=i, dtype=dtype) for i, h in enumerate((4, 2, 2)))
    clean = ops.ragged_attention(q, k, v, ints(*at), window=window)
    rows = torch.tensor([a + w for a, w in zip(at, where)], device="cuda")
    q[rows, :, 5] = float("nan")
    got = ops.ragged_attention(q, k, v, ints(*at), window=window)
    assert got[rows].isnan().all()
    others = torch.ones(at[-1], dtype=torch.bool, device="cuda").index_fill_(0, rows, False)
    assert torch.equal(got[others], clean[others])


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("size", [1.0, 1e3, 1e5, 1e6])
def test_ragged_fp16_gradients_of_large_scores(dim, size):
    """fp16: gradients of scores beyond 65504 whose products with small keys and queries are within the type, beside rows of ordinary
    size. The bound's last term: weights of 2^26 times the type's smallest half step, 2^-25, in rows that need the wider range."""
    lens = [70, 5, 300, 131]
    at = plain.starts(lens)
    q, k, v, do = (rnd(at[-1], h, dim, seed=i, dtype=FP16) for i, h in enumerate((4, 2, 2, 4)))
    large = slice(at[2], at[3])
    k[large] *= 2.0 ** -10
    q[large] *= 2.0 ** -10
    v[large] *= size ** 0.5
    do[at[2] + 1:at[3]] *= size ** 0.5
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.ragged_attention(*leaves, ints(*at)), leaves, do)
    (_, (dq, eq), (dk, ek), (dv, ev)) = plain.ragged(q, k, v, at, at, None, dim ** -0.5, do)
    room = torch.zeros(at[-1], dtype=torch.float64, device="cuda")
    room[large] = 2.0 * lens[2] * 2 * dim ** -0.5 if size > 1 else 0.0          # two heads' sums of up to 300 weights off by up to 2
    most = lambda t: room[:, None, None] * t[large].double().abs().amax()  # noqa: E731
    for got, w, b in zip(grads, (dq, dk, dv), (eq + most(k), ek + most(q), ev)):
        assert w.abs().max() < 60000
        plain.near(got, w, b)


def test_ragged_under_function_transforms():
    """Forward-mode derivatives and ``torch.func.grad`` against those of the double-precision formula; never a silent zero. Sums are 32-bit, the
    result is rounded to fp16: half a step is 2^-11 of a value."""
    at = [0, 13, 40]
    q, k, v, t = (rnd(40, h, 16, seed=i, dtype=FP16) for i, h in enumerate((4, 2, 2, 4)))

    def formula(x, kk, vv):
        return torch.cat([torch.cat([plain.softmax(x[a:z, h] @ kk[a:z, h // 2].T / 4, plain.visible(z - a, z - a, None, "cuda")) @ vv[a:z, h // 2]
                                     for h in range(4)], 1).unflatten(1, (4, 16)) for a, z in zip(at, at[1:])])

    _, want = torch.func.jvp(lambda x: formula(x, k.double(), v.double()), (q.double(),), (t.double(),))
    _, got = torch.func.jvp(lambda x: ops.ragged_attention(x, k, v, ints(*at)), (q,), (t,))
    assert want.abs().max() > 0.1 and (got.double() - want).abs().max() < 2.0 ** -10 * max(1.0, want.abs().max().item())
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, t)
        tangent = torch.autograd.forward_ad.unpack_dual(ops.ragged_attention(dual, k, v, ints(*at))).tangent
    assert torch.equal(tangent, got)
    want = torch.func.grad(lambda x: (formula(x, k.double(), v.double()) * t.double()).sum())(q.double())
    got = torch.func.grad(lambda x: (ops.ragged_attention(x, k, v, ints(*at)).float() * t.float()).sum())(q)
    assert (got.double() - want).abs().max() < 2.0 ** -10 * max(1.0, want.abs().max().item())


def test_ragged_gradients_have_the_strides_that_a_trace_is_told():
    """Layouts of operands, neighbours in memory or only alike: what the kernel returns is laid out as its shape implementation says."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    heads, kv, dim, rows, at = 4, 2, 64, 30, ints(0, 13, 30)
    wide = (heads + 2 * kv) * dim
    x = rnd(rows, wide, dtype=BF16)
    q, k, v = (t.view(rows, -1, dim) for t in x.split([heads * dim, kv * dim, kv * dim], 1))
    other = torch.empty(rows, wide, dtype=BF16, device="cuda")[:, 64:64 + kv * dim].view(rows, kv, dim).copy_(k)       # alike, elsewhere
    odd = torch.empty(rows * wide + 1, dtype=BF16, device="cuda")[1:].view(rows, wide)[:, :kv * dim].view(rows, kv, dim).copy_(k)     # between 16-byte boundaries
    cases = [(q, k, v), (q.contiguous(), k, v), (q, k.contiguous(), v), (q, other, v), (q, odd, v), (q, v, k), (q.transpose(0, 1).contiguous().transpose(0, 1), k, v)]
    grads = []
    for a, b, c in cases:
        o, lse = _op("ragged_fwd")(a, b, c, at, at, 0.125, 0, True)
        args = (torch.ones_like(o), a, b, c, o, lse, at, at)
        real = _op("ragged_bwd")(*args, 0.125, 0)
        with FakeTensorMode() as mode:
            told = _op("ragged_bwd")(*(mode.from_tensor(t) for t in args), 0.125, 0)
        for r, t in zip(real, told):
            assert r.shape == t.shape and r.stride() == t.stride()
        grads.append(real)
    for i in (1, 2, 3, 4, 6):           # the same operands in other places
        for r, t in zip(grads[i], grads[0]):
            assert torch.equal(r, t)


def test_ragged_traced_training_step_of_a_joint_projection():
    """Forward and backward as one traced graph, which is told shapes and strides only, against the same step untraced."""
    heads, kv, dim, rows, at = 4, 2, 64, 48, ints(0, 13, 48)
    x, w, do = rnd(rows, 96, seed=1, dtype=BF16), rnd(96, (heads + 2 * kv) * dim, seed=2, dtype=BF16, scale=0.1), rnd(rows, heads * dim, seed=3, dtype=BF16)

    def step(x, w, do):
        q, k, v = (t.view(rows, -1, dim) for t in (x @ w).split([heads * dim, kv * dim, kv * dim], 1))
        o = ops.ragged_attention(q, k, v, at).flatten(1)
        return torch.autograd.grad(o, w, do)[0]

    from torch.fx.experimental.proxy_tensor import make_fx
    leaf = w.clone().requires_grad_()
    want = step(x, leaf, do)
    traced = make_fx(step, tracing_mode="fake", _allow_non_fake_inputs=True)(x, leaf, do)
    assert any("ragged_bwd" in str(n.target) for n in traced.graph.nodes)
    assert torch.equal(traced(x, leaf, do), want)


def test_ragged_in_32_bits_on_the_gpu():
    """Computed sequence by sequence in PyTorch: as on the CPU, to 128 terms of 2^-24 twice over, forward and backward."""
    at = [0, 5, 5, 90, 131]
    made = [rnd(140, h, 24, seed=i) for i, h in enumerate((4, 2, 2, 4))]
    both = []
    for dev in ("cuda", "cpu"):
        leaves = [t.to(dev, copy=True).requires_grad_() for t in made[:3]]
        o = ops.ragged_attention(*leaves, torch.tensor(at, dtype=torch.int32, device=dev), window=40)
        both.append([t.cpu() for t in (o.detach(), *torch.autograd.grad(o, leaves, made[3].to(dev)))])
    for a, b in zip(*both):
        assert (a - b).abs().max() <= plain.SMALL * max(1.0, b.abs().max().item()) * 8          # sums of up to 8 such terms' size


# ------------------------------------------------------------------------------------------------------------------ pages
@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_paged_attention_scores_that_are_infinite_or_no_number(rows, dtype, dim):
    """Bad keys at each place of a batch. All scores minus infinity, one plus infinity or one no number: NaN. Minus infinity beside finite
    scores: as without that key. Nothing to see: zeros."""
    length, page = 150, 16
    columns = -(-length // page)
    table = torch.arange(rows * columns, dtype=torch.int32, device="cuda").view(rows, columns)
    q = rnd(rows, 4, dim, seed=1, dtype=dtype)
    q[:, :, 3] = 1.0
    kp, vp = (rnd(rows * columns, 2, page, dim, seed=i, dtype=dtype) for i in (2, 3))
    lens = torch.full((rows,), length, dtype=torch.int32, device="cuda")
    clean = ops.paged_attention(q, kp, vp, table, lens)
    for place in (0, 5, 15, 16, 63, 64, 149):
        for what in (float("nan"), float("inf"), float("-inf")):
            bad = kp.clone()
            bad[table[:, place // page].long(), :, place % page, 3] = what
            got = ops.paged_attention(q, bad, vp, table, lens)
            if what != float("-inf"):
                assert got.isnan().all(), (place, what)
                continue
            b = rows - 1
            k, v = plain.held(kp, None, table, b, length), plain.held(vp, None, table, b, length)
            keep = [j for j in range(length) if j != place]
            u = plain.U[dtype]
            for h in range(4):
                p = torch.softmax(k[keep, h // 2] @ q[b, h].double() * dim ** -0.5, 0)
                w, e = p @ v[keep, h // 2], p @ v[keep, h // 2].abs()
                assert ((got[b, h].double() - w).abs() <= (u + plain.SMALL) * e + u * w.abs() + 2.0 ** -24).all()
    kp[..., 3] = float("-inf")
    for n in (1, 17, 150):
        for window in (None, 3):
            lens.fill_(n)
            lens[0] = 0 if rows > 1 else n
            got = ops.paged_attention(q, kp, vp, table, lens, window=window)
            assert got[rows > 1:].isnan().all() and (rows == 1 or not got[0].any())
    assert clean.isfinite().all()
