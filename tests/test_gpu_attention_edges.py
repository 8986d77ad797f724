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


def _norm_inputs(dev):
    from wallx_mi355 import workloads as wl

    q, k = (torch.randn(2, h, 20, 128, device=dev).to(torch.bfloat16) for h in (4, 2))
    w = torch.ones(128, dtype=torch.bfloat16, device=dev)
    pos, freq, section = torch.arange(20, device=dev).expand(3, 2, 20).contiguous(), wl.text_inv_freq(128).to(dev), list(wl.MROPE_SECTION)
    table = ops.multimodal_rope_table(pos, freq, section)
    return q, k, w, lambda q, k, wq, wk: ops.qk_norm_rope_from_table(q, k, wq, wk, table, section), lambda q, k, wq, wk: ops.qk_norm_rope_from_positions(q, k, wq, wk, pos, freq, section)


@pytest.mark.parametrize("leaf", [False, True])
def test_forward_mode_is_refused(dev, host, leaf):
    """A tangent is never dropped without a word, whether its tensor requires grad or not, and neither under no_grad."""
    from torch.autograd import forward_ad as fw

    q, k, w, from_table, from_positions = _norm_inputs(dev)
    cache = ops.quantized_kv_cache(2, 2, 40, 128, dev)
    start = torch.zeros(2, dtype=torch.int32, device=dev)
    calls = [lambda d: from_table(d(q), k, w, w), lambda d: from_table(q, k, w, d(w)), lambda d: from_positions(q, d(k), w, w),
             lambda d: ops.attention(d(q), k, k), lambda d: ops.attention(q, k, d(k), causal=True), lambda d: ops.cached_attention(d(q), *cache),
             lambda d: ops.kv_cache_write(k, d(k), *cache, start)]
    before = [t.view(torch.uint8).clone() if t.dtype == torch.float8_e4m3fn else t.clone() for t in cache]
    for i, call in enumerate(calls):
        with fw.dual_level():
            dual = lambda t: fw.make_dual(t.detach().clone().requires_grad_(leaf), torch.ones_like(t))  # noqa: E731
            with pytest.raises(RuntimeError, match="forward-mode|forward AD|not differentiable"):
                call(dual)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call(dual)
            call(lambda t: t)  # the level alone is no reason
        if i < 6:
            assert all(torch.equal(a, b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b) for a, b in zip(before, cache))


def test_graphs_of_gradients(dev, host):
    """create_graph=True is for what is differentiated twice: the ops' gradients come out the same, other paths' second derivatives are right, and
    the ops' own are refused where they are asked for."""
    q, k, w, from_table, from_positions = _norm_inputs(dev)
    v = torch.randn_like(k)
    for op, args in ((lambda *a: (ops.attention(*a, causal=True),), (q, k, v)), (from_table, (q, k, w, w)), (from_positions, (q, k, w, w))):
        for transposed in (False, True):  # (what is copied first goes another way)
            leaves = [t.detach().clone().requires_grad_() for t in args]
            used = [t.transpose(-1, -2).contiguous().transpose(-1, -2) if transposed and t.dim() == 4 else t for t in leaves]
            out = op(*used)
            do = [torch.randn_like(y) for y in out]
            want = torch.autograd.grad(out, leaves, do, retain_graph=True)
            got = torch.autograd.grad(out, leaves, do, create_graph=True)
            assert all(torch.equal(a, b) for a, b in zip(want, got))
            # a penalty beside the op: its own second derivative
            x = torch.tensor(3.0, device=dev, requires_grad=True)
            total = sum(y.float().sum() for y in op(*used)) + x ** 3
            (gx,) = torch.autograd.grad(total, x, create_graph=True)
            (ggx,) = torch.autograd.grad(gx, x)
            assert float(ggx) == 18.0
            total.backward(create_graph=True)
            assert float(x.grad) == 27.0 and all(torch.isfinite(t.grad).all() for t in leaves)
            for t in (*leaves, x):
                t.grad = None
            # the op's: wherever a path leads through it, also beside another one, and from the gradient that came in
            for leaf in leaves:
                got = torch.autograd.grad(op(*used), leaves, do, create_graph=True)
                with pytest.raises(RuntimeError, match="not differentiable|differentiate twice"):
                    torch.autograd.grad(sum(g.float().square().sum() for g in got) + (leaf.float() ** 2).sum(), leaf)
            sums = [d.clone().requires_grad_() for d in do]
            got = torch.autograd.grad(op(*used), leaves, sums, create_graph=True)
            with pytest.raises(RuntimeError, match="not differentiable|differentiate twice"):
                got[0].float().sum().backward()


def test_the_most_sequences(dev):
    """As many sequences of one token as a launch has workgroups for, and one more, which is refused (in front of any launch)."""
    most = 2 ** 24 - 1
    x = torch.arange(most + 1, device=dev, dtype=torch.int32).bitwise_and(2047).to(torch.float16).view(-1, 1, 1, 1).expand(-1, 1, 1, 64).contiguous()
    start = torch.zeros(most + 1, dtype=torch.int32, device=dev)
    cache = ops.quantized_kv_cache(most + 1, 1, 1, 64, dev)
    with pytest.raises(RuntimeError, match="too many"):
        ops.kv_cache_write(x, x, *cache, start)
    with pytest.raises(RuntimeError, match="too many"):
        ops.attention(x, x, x)
    with pytest.raises(RuntimeError, match="too many"):
        ops.cached_attention(x, *cache)
    assert not any(t.view(torch.uint8).any() for t in cache)
    x, start, cache = x[:most], start[:most], ops.quantized_kv_cache(most, 1, 1, 64, dev)
    # (scores of up to 2047 * 2047 * 64 / 8 = 2^25 natural units, 4.8e7 powers of two, where fp32 numbers are 4 apart: the only probability is
    # 2^-2 to 2^2, and rounded to fp16 while the sum of them is not: half a step of it, and half a step of the result)
    assert bool(((ops.attention(x, x, x).float() - x.float()).abs() <= 2.0 ** -10 * x.float()).all())
    ops.kv_cache_write(x, x, *cache, start)
    # (a row of one value: its code is 448, its scale a 448th of it to fp32)
    assert float((ops.cached_attention(x, *cache).float() - x.float()).abs().max()) <= 2048 * 2.0 ** -11
    del cache
    most = 2 ** 22 - 1  # (the backward plans a pair with 1024 threads)
    leaf = x[:most].clone().requires_grad_()
    (g,) = torch.autograd.grad(ops.attention(leaf, leaf, leaf, scale=2.0 ** -20), leaf, x[:most])  # (scores below 2^9, as exact as they come)
    assert torch.equal(g, x[:most])
    leaf = x[:most + 1].clone().requires_grad_()
    out = ops.attention(leaf, leaf, leaf)
    with pytest.raises(RuntimeError, match="too many"):
        torch.autograd.grad(out, leaf, x[:most + 1])
