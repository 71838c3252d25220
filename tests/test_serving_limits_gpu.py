"""Serving operators where their inputs are at a limit: infinities and what is no number, rows of a cluster, borders of a sum, 16-bit
ranges. The statements in 64 bits and their bounds are ``plain_serving``'s."""
import pytest
import torch

from oslo_b200 import ops

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
