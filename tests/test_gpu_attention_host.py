"""The attention, norm and cache ops through the native host module and through the general path give the same bits, and what
autograd sees of them: in-place writes, saved tensors, double backward, inference mode, no gradients wanted."""

import pytest
import torch

from wallx_mi355 import _lib, workloads as wl
from wallx_mi355.fusions import ops

pytestmark = pytest.mark.gpu
SECTION = list(wl.MROPE_SECTION)


def _inputs(dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    make = lambda h: torch.randn(2, 40, h, 128, generator=g, device=dev).to(torch.bfloat16).transpose(1, 2)  # noqa: E731
    return make(8), make(2), make(2), make(8), make(2)


def _everything(dev):
    q, k, v, gq, gk = _inputs(dev)
    w = torch.linspace(0.5, 1.5, 128, device=dev).to(torch.bfloat16)
    pos = torch.arange(40, device=dev).expand(3, 2, 40).contiguous()
    freq = wl.text_inv_freq(128).to(dev)
    table = ops.multimodal_rope_table(pos, freq, SECTION)
    ranges = ops.attention_key_ranges(torch.arange(40, device=dev).expand(2, 40) > 30)
    lengths = torch.tensor([40, 33], dtype=torch.int32, device=dev)
    out = []
    for op in (lambda *a: ops.qk_norm_rope_from_table(*a, table, SECTION), lambda *a: ops.qk_norm_rope_from_positions(*a, pos, freq, SECTION, eps=1e-5, layout="csrc")):
        leaves = [t.detach().requires_grad_() for t in (q, k, w, w)]
        y = op(*leaves)
        out += [*y, *torch.autograd.grad(y, leaves, (gq, gk)), *op(q, k, w, w)]
    for kw in (dict(causal=True), dict(key_ranges=ranges), dict(key_lengths=lengths, scale=0.3)):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        y = ops.attention(*leaves, **kw)
        out += [y, *torch.autograd.grad(y, leaves, gq), ops.attention(q, k, v, **kw)]
    cache = ops.quantized_kv_cache(2, 2, 64, 128, dev)
    ops.kv_cache_write(k, v, *cache, lengths - 30, lengths=lengths)
    out += [t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in cache]
    out += [ops.cached_attention(q, *cache, key_lengths=lengths, causal=True), ops.cached_attention(q, *cache, key_ranges=ranges, scale=0.2)]
    return [t.detach() for t in out]


def test_both_paths_give_the_same(dev, monkeypatch):
    fast = _everything(dev)
    monkeypatch.setattr(_lib, "_host", _lib._NoHost)
    for i, (a, b) in enumerate(zip(fast, _everything(dev))):
        assert torch.equal(a, b) and a.stride() == b.stride(), i


@pytest.mark.parametrize("native_host", [True, False])
def test_autograd(dev, monkeypatch, native_host):
    if not native_host:
        monkeypatch.setattr(_lib, "_host", _lib._NoHost)
    q, k, v, gq, _ = _inputs(dev, 1)
    leaf = q.detach().clone().requires_grad_()
    # one gradient wanted: the others are not made
    out = ops.attention(leaf, k, v, causal=True)
    assert out.requires_grad and not out._is_view()
    (dq,) = torch.autograd.grad(out, leaf, gq, retain_graph=True)
    # what a caller writes into the result in place is an autograd operation like any other ...
    scaled = ops.attention(leaf, k, v, causal=True) * 1
    scaled.mul_(2)
    (twice,) = torch.autograd.grad(scaled, leaf, gq)
    assert torch.equal(twice, torch.autograd.grad(ops.attention(leaf, k, v, causal=True), leaf, gq * 2)[0])
    # ... and what the backward needs and finds overwritten is refused
    out = ops.attention(leaf, k, v, causal=True)
    out.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, leaf, gq)
    kk = k.clone()
    out = ops.attention(leaf, kk, v, causal=True)
    kk.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, leaf, gq)
    # no second derivative
    out = ops.attention(leaf, k, v, causal=True)
    with pytest.raises(RuntimeError, match="differentia|does not require grad"):
        (g1,) = torch.autograd.grad(out, leaf, gq, create_graph=True)
        torch.autograd.grad(g1.sum(), leaf)
    # a gradient in another order, and one value for all
    out = ops.attention(leaf, k, v, causal=True)
    odd = gq.transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(torch.autograd.grad(out, leaf, odd, retain_graph=True)[0], dq)
    one = torch.ones((), dtype=torch.bfloat16, device=dev).expand(gq.shape)
    assert torch.equal(torch.autograd.grad(out, leaf, one, retain_graph=True)[0], torch.autograd.grad(out, leaf, torch.ones_like(gq))[0])
    # an unused result of the norm
    w = torch.ones(128, dtype=torch.bfloat16, device=dev, requires_grad=True)
    table = ops.multimodal_rope_table(torch.zeros(3, 2, 40, dtype=torch.int64, device=dev), wl.text_inv_freq(128).to(dev), SECTION)
    y, _ = ops.qk_norm_rope_from_table(leaf, k, w, w, table, SECTION)
    dl, dw = torch.autograd.grad(y, (leaf, w), gq)
    assert torch.isfinite(dl).all() and torch.isfinite(dw).all()
    # neither a graph where none is wanted, nor gradients where there are none
    with torch.no_grad():
        assert not ops.attention(leaf, k, v).requires_grad
    cache = ops.quantized_kv_cache(2, 2, 64, 128, dev)
    start = torch.zeros(2, dtype=torch.int32, device=dev)
    with pytest.raises(RuntimeError, match="not differentiable"):
        ops.cached_attention(leaf, *cache)
    with pytest.raises(RuntimeError, match="not differentiable"):
        ops.kv_cache_write(leaf[:, :2], leaf[:, :2], *cache, start)
    before = [t._version for t in cache]
    ops.kv_cache_write(k, v, *cache, start)
    assert all(t._version > n for t, n in zip(cache, before))
    with torch.inference_mode():
        inner = ops.quantized_kv_cache(2, 2, 64, 128, dev)
        ops.kv_cache_write(k, v, *inner, start)
        assert torch.equal(ops.cached_attention(q, *inner), ops.cached_attention(q, *cache))


@pytest.mark.parametrize("native_host", [True, False])
def test_refusals(dev, monkeypatch, native_host):
    if not native_host:
        monkeypatch.setattr(_lib, "_host", _lib._NoHost)
    q, k, v, _, _ = _inputs(dev, 2)
    r = torch.zeros(2, 40, 2, dtype=torch.int32, device=dev)
    for args, kw, what in (((q, k, v[:, :1]), {}, "inconsistent"), ((q, k[:1], v[:1]), {}, "inconsistent"), ((q, k.float(), v), {}, "one dtype"),
                           ((q.float(), k.float(), v.float()), {}, "BFloat16 or Half"), ((q[:, :3], k, v), {}, "no multiple"),
                           ((q[..., :96], k[..., :96], v[..., :96]), {}, "64, 80 or 128"), ((q[0], k, v), {}, "B, H, S, D"),
                           ((q, k, v), dict(key_ranges=r[:, :3]), "key_ranges"), ((q, k, v), dict(key_ranges=r.long()), "key_ranges"),
                           ((q, k, v), dict(key_lengths=r[0, :, 0]), "key_lengths"), ((q, k, v), dict(key_ranges=r.cpu()), "CUDA"),
                           ((q, k, v), dict(scale=-1.0), "scale"), ((q, k, v), dict(scale=float("nan")), "scale"), ((q, k.cpu(), v), {}, "CPU")):
        with pytest.raises(RuntimeError, match=what):
            ops.attention(*args, **kw)
    cache = ops.quantized_kv_cache(2, 2, 64, 128, dev)
    start = torch.zeros(2, dtype=torch.int32, device=dev)
    for args, what in (((k, v, cache[0].float(), *cache[1:], start), "k_cache"), ((k, v, *cache[:2], cache[2][:, :1], cache[3], start), "k_scale"),
                       ((k[:, :1], v[:, :1], *cache, start), "differ in batch"), ((k, v, *cache, start.long()), "start"), ((k, v, *cache, start[:1]), "start"),
                       ((k.float(), v.float(), *cache, start), "BFloat16 or Half"), ((k, v[:, :, :3], *cache, start), "one shape"),
                       ((k, v, cache[0].transpose(0, 1), *cache[1:], start), "k_cache")):
        with pytest.raises(RuntimeError, match=what):
            ops.kv_cache_write(*args)
    with pytest.raises(RuntimeError, match="batch and head size"):
        ops.cached_attention(q[:1], *cache)
    w = torch.ones(128, dtype=torch.bfloat16, device=dev)
    pos, freq = torch.zeros(3, 2, 40, dtype=torch.int64, device=dev), wl.text_inv_freq(128).to(dev)
    table = ops.multimodal_rope_table(pos, freq, SECTION)
    for args, kw, what in (((q, k, w[:64], w, table, SECTION), {}, "q_weight"), ((q, k, w.float(), w, table, SECTION), {}, "one dtype"),
                           ((q, k, w, w, table[:3], SECTION), {}, "table"), ((q, k, w, w, table, SECTION), dict(layout="csrc"), "table"),
                           ((q, k, w, w, table, SECTION), dict(layout="no"), "layout"), ((q, k[:, :, :3], w, w, table, SECTION), {}, "inconsistent"),
                           ((q, k, w, w, table, [64, 0]), {}, "3 integers"), ((q, k, w, w, table, SECTION), dict(eps=-1.0), "eps")):
        with pytest.raises(RuntimeError, match=what):
            ops.qk_norm_rope_from_table(*args, **kw)
    with pytest.raises(RuntimeError, match="position_ids"):
        ops.qk_norm_rope_from_positions(q, k, w, w, pos[:, :1], freq, SECTION)
    with pytest.raises(RuntimeError, match="inv_freq"):
        ops.qk_norm_rope_from_positions(q, k, w, w, pos, freq[:5], SECTION)
