"""Calls of the attention ops at the edges of what their documentation allows, through the native host module and without it."""

import pytest
import torch

from wallx_mi355 import _lib
from wallx_mi355.fusions import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[True, False], ids=["native host", "python host"])
def host(request, monkeypatch):
    if not request.param:
        monkeypatch.setattr(_lib, "_host", _lib._NoHost)


@pytest.mark.parametrize("Sq", [0, 1, 70])
@pytest.mark.parametrize("Sk", [1, 300, 5000])
def test_no_query_heads(dev, host, Sq, Sk):
    """Nothing reads the keys: their gradients are zeros, every one of them."""
    for D, dtype in ((64, torch.bfloat16), (128, torch.float16)):
        q = torch.empty(3, 0, Sq, D, dtype=dtype, device=dev, requires_grad=True)
        k, v = (torch.randn(3, 2, Sk, D, device=dev).to(dtype).requires_grad_() for _ in range(2))
        out = ops.attention(q, k, v, causal=True)
        assert out.shape == q.shape
        junk = [torch.full((3, 2, Sk, D), float("nan"), dtype=dtype, device=dev) for _ in range(8)]  # what the gradients' memory may hold
        del junk
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), torch.empty_like(out))
        assert dq.shape == q.shape and torch.equal(dk, torch.zeros_like(k)) and torch.equal(dv, torch.zeros_like(v))
