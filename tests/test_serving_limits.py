"""Serving operators at the limits of what they are given, on the CPU."""
import pytest
import torch

import oslo_b200 as ob
from oslo_b200 import ops
from oslo_b200.generation import PagedKVCache
from oslo_b200.ops.cuda_ops import _op


def rnd(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed + sum(shape))).to(dtype)


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.mark.parametrize("joint", [True, False])
def test_ragged_gradients_of_a_trace_have_their_strides(joint):
    """Gradients of slices of one projection are slices of one tensor, also where only shapes are traced; others are contiguous."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    if ops.load_ext() is None:
        pytest.skip("the extension is not built")
    heads, kv, dim, rows = 4, 2, 64, 30
    with FakeTensorMode():
        x = torch.empty(rows, (heads + 2 * kv) * dim, dtype=torch.bfloat16, device="cuda")
        q, k, v = (t.view(rows, -1, dim) for t in x.split([heads * dim, kv * dim, kv * dim], 1))
        if not joint:
            k = k.contiguous()
        at = torch.empty(4, dtype=torch.int32, device="cuda")
        do, o, lse = torch.empty_like(q), torch.empty_like(q), torch.empty(rows, heads, device="cuda")
        got = _op("ragged_bwd")(do, q, k, v, o, lse, at, at, 0.125, 0)
        for g, t in zip(got, (q, k, v)):
            assert g.shape == t.shape and g.dtype == t.dtype
            assert g.stride() == (t.stride() if joint else (t.size(1) * dim, dim, 1))


@pytest.mark.parametrize("what", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ragged_statement_keeps_sequences_apart(what, dtype):
    """What is no number in one sequence, or in rows of none, leaves the others as they are - forward and backward."""
    at = [2, 9, 20, 33]
    q, k, v, do = (rnd(40, h, 8, seed=i, dtype=dtype) for i, h in enumerate((4, 2, 2, 4)))
    clean = [t.clone().requires_grad_() for t in (q, k, v)]
    o1 = ops.ragged_attention(*clean, ints(*at))
    g1 = torch.autograd.grad(o1, clean, do)
    for t in (q, k, v, do):
        t[:2] = t[9:20] = t[33:] = what
    bad = [t.clone().requires_grad_() for t in (q, k, v)]
    o2 = ops.ragged_attention(*bad, ints(*at))
    g2 = torch.autograd.grad(o2, bad, do)
    for a, b in zip((o1, *g1), (o2, *g2)):
        assert torch.equal(a[2:9], b[2:9]) and torch.equal(a[20:33], b[20:33])
        assert not b[:2].any() and not b[33:].any()
    assert o2[9:20].isnan().all()


def test_ragged_statement_without_rows_or_keys():
    for rows, keys, starts, key_starts in ((0, 5, (0, 0), (0, 5)), (5, 0, (0, 5), (0, 0)), (5, 4, (0, 0, 0), (0, 2, 4)), (3, 4, (0, 1, 3), (0, 4, 4))):
        leaves = [rnd(rows, 4, 8, seed=1).requires_grad_(), rnd(keys, 2, 8, seed=2).requires_grad_(), rnd(keys, 2, 8, seed=3).requires_grad_()]
        o = ops.ragged_attention(*leaves, ints(*starts), ints(*key_starts))
        assert o.shape == leaves[0].shape and o.isfinite().all() and not o[1:].any()
        assert all(g.isfinite().all() for g in torch.autograd.grad(o.sum(), leaves))


def tiny(cls=None):
    torch.manual_seed(0)
    return (cls or ob.GPT2LMHeadModel)(ob.GPT2Config(vocab_size=61, n_positions=64, n_embd=32, n_layer=2, n_head=2)).eval()


def test_generate_calls_overridden_steps_as_it_did():
    """Subclasses that were written before ``min_p`` and ``fused_sampling`` are not handed what they do not know."""
    class Older(ob.GPT2LMHeadModel):
        @staticmethod
        def _get_logits_warper(top_k, top_p, temperature, num_beams):
            return ob.GPT2LMHeadModel._get_logits_warper(top_k, top_p, temperature, num_beams)

        def sample(self, input_ids, logits_processor=None, stopping_criteria=None, logits_warper=None, pad_token_id=None, eos_token_id=None,
                   output_scores=False, return_dict_in_generate=False, synced_gpus=False, **model_kwargs):
            return super().sample(input_ids, logits_processor, stopping_criteria, logits_warper, pad_token_id, eos_token_id, output_scores,
                                  return_dict_in_generate, synced_gpus, **model_kwargs)

    ids = torch.arange(6).view(2, 3)
    outs = []
    for model in (tiny(), tiny(Older)):
        torch.manual_seed(3)
        outs.append(model.generate(ids, do_sample=True, max_length=12, top_k=9))
    assert outs[0].tolist() == outs[1].tolist()


@pytest.mark.parametrize("missing", ["temperature", "top_k", "top_p"])
def test_fused_sampling_with_a_setting_that_the_config_leaves_out(missing):
    model = tiny()
    setattr(model.config, missing, None)
    ids = torch.arange(6).view(2, 3)
    assert model.generate(ids, do_sample=True, max_length=9).shape == (2, 9)
    assert model.generate(ids, do_sample=True, max_length=9, fused_sampling=True).shape == (2, 9)


def test_fused_sampling_whatever_the_default_type():
    model = tiny()
    torch.set_default_dtype(torch.bfloat16)
    try:
        assert model.generate(torch.arange(6).view(2, 3), do_sample=True, max_length=9, fused_sampling=True).shape == (2, 9)
    finally:
        torch.set_default_dtype(torch.float32)


@pytest.mark.parametrize("bad", [dict(dtype=torch.float32), dict(dtype=torch.float32, quantised=True), dict(dim=20), dict(dim=264), dict(dim=24, quantised=True)])
def test_a_cache_that_the_kernels_cannot_fill_is_refused_when_it_is_made(bad):
    with pytest.raises(ValueError, match="GPU"):
        PagedKVCache(**dict(dict(layers=1, pages=4, page=8, heads=2, dim=64, rows=2, device="cuda"), **bad))
    PagedKVCache(**dict(dict(layers=1, pages=4, page=8, heads=2, dim=64, rows=2, device="cpu"), **bad))


def test_a_row_holds_max_length_tokens_and_no_more():
    cache = PagedKVCache(layers=1, pages=9, page=4, heads=1, dim=16, rows=2, dtype=torch.float32, max_length=10)
    cache.extend([9, 3])
    with pytest.raises(RuntimeError, match="10"):
        cache.extend([2, 0])
    assert cache.lengths.tolist() == [9, 3] and cache.free_pages == 5
    cache.extend([1, 7])
    assert cache.lengths.tolist() == [10, 10]
    with pytest.raises(ValueError):
        PagedKVCache(layers=1, pages=9, page=4, heads=1, dim=16, rows=2, max_length=0)


def test_pages_are_handed_out_on_the_host_whatever_the_default_device():
    torch.set_default_device("meta")
    try:
        cache = PagedKVCache(layers=1, pages=6, page=4, heads=1, dim=16, rows=2, dtype=torch.float32, device="cpu")
        cache.extend([5, 1])
        cache.release(0)
    finally:
        torch.set_default_device(None)
    assert cache.lengths.tolist() == [0, 1] and cache.free_pages == 5
