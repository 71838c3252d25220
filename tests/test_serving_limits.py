"""Serving operators at the limits of what they are given, on the CPU."""
import pytest
import torch

from oslo_b200 import ops


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
        got = torch.ops.oslo_b200.ragged_bwd(do, q, k, v, o, lse, at, at, 0.125, 0)
        for g, t in zip(got, (q, k, v)):
            assert g.shape == t.shape and g.dtype == t.dtype
            assert g.stride() == (t.stride() if joint else (t.size(1) * dim, dim, 1))
