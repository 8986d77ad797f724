"""The norm, the attention and the cache as a decoder runs them one after another: a training step from the hidden states to the
gradients, a prefill and its denoise steps over the quantised cache, the prefill harness on them; captured, on two streams, under
checkpointing and with tensors saved on the host."""

import pytest
import torch
import torch.nn.functional as F

from test_gpu_attention import check, reference, visible
from test_gpu_harness import _ref_forward
from wallx_mi355 import workloads as wl
from wallx_mi355.fusions import ops

pytestmark = pytest.mark.gpu
SECTION = list(wl.MROPE_SECTION)
B, S, H, HQ, HKV, D = 2, 90, 256, 8, 2, 128


def parameters(dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    make = lambda *shape, by=1.0: (torch.randn(*shape, generator=g, device=dev) * by).to(torch.bfloat16)  # noqa: E731
    x, wqkv, wo = make(B, S, H), make((HQ + 2 * HKV) * D, H, by=H ** -0.5), make(H, HQ * D, by=(HQ * D) ** -0.5)
    wq, wk = (1 + 0.2 * torch.randn(D, generator=g, device=dev)).to(torch.bfloat16), (1 + 0.2 * torch.randn(D, generator=g, device=dev)).to(torch.bfloat16)
    return x, wqkv, wo, wq, wk


def positions(dev, start=0, n=S):
    return (start + torch.arange(n, device=dev)).expand(3, B, n).contiguous()


def project(x, wqkv, wq, wk, pos, freq):
    b, s = x.shape[:2]
    q, k, v = (t.view(b, s, -1, D).transpose(1, 2) for t in F.linear(x, wqkv).split([HQ * D, HKV * D, HKV * D], -1))
    q, k = ops.qk_norm_rope_from_positions(q, k, wq, wk, pos, freq, SECTION)
    return q, k, v


def layer(x, wqkv, wo, wq, wk, pos, freq, ranges):
    q, k, v = project(x, wqkv, wq, wk, pos, freq)
    return F.linear(ops.attention(q, k, v, ranges).transpose(1, 2).reshape(x.size(0), x.size(1), HQ * D), wo)


def plain_layer(x, wqkv, wo, wq, wk, pos, freq, see):
    b, s = x.shape[:2]
    q, k, v = (t.reshape(b, s, -1, D).transpose(1, 2) for t in (x @ wqkv.T).split([HQ * D, HKV * D, HKV * D], -1))
    a = pos.double()[..., None] * freq.double()
    parts = torch.cat((a, a), -1).split(SECTION * 2, -1)
    a = torch.cat([p[i % 3] for i, p in enumerate(parts)], -1)[:, None]

    def turned(t, w):
        t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * w
        return t * a.cos() + torch.cat((-t[..., D // 2:], t[..., :D // 2]), -1) * a.sin()

    q, k = turned(q, wq), turned(k, wk)
    k, v = k.repeat_interleave(HQ // HKV, 1), v.repeat_interleave(HQ // HKV, 1)
    p = torch.softmax((q @ k.transpose(-1, -2) * D ** -0.5).masked_fill(~see, float("-inf")), -1)
    return (p @ v).transpose(1, 2).reshape(b, s, HQ * D) @ wo.T


def types_of(dev):
    types = torch.zeros(B, S, dtype=torch.bool, device=dev)
    types[0, S - 16:], types[1, 40:56] = True, True
    return types


def test_training_step(dev):
    """Against autograd of the plain layer in 64 bits.  Between the inputs and a gradient lie at most ten roundings to bfloat16
    (projection, norm with rotation, probabilities, attention's output, the o projection's gradient, slopes, attention's and the norm's
    gradients, the projection's gradient), each of at most 2^-8 of the values rounded; a score, |q| |k| / sqrt(D) = 11.3 at most, moves by the
    roundings of 128 products, 2^-8 sqrt(2) in the mean, as one rounding of a probability does.  So 12 * 2^-8 of a gradient's
    length; what is wired wrongly is off by its whole length."""
    args = parameters(dev)
    freq, pos, types = wl.text_inv_freq(D).to(dev), positions(dev), types_of(dev)
    ranges = ops.attention_key_ranges(types)
    see = visible(B, S, S, dev, ranges)
    g = torch.Generator(device=dev).manual_seed(1)
    do = torch.randn(B, S, H, generator=g, device=dev).to(torch.bfloat16)
    leaves = [t.clone().requires_grad_() for t in args]
    out = layer(*leaves, pos, freq, ranges)
    got = (out.detach(), *torch.autograd.grad(out, leaves, do))
    plain = [t.double().cpu().requires_grad_() for t in args]
    ref = plain_layer(*plain, pos.cpu(), freq.cpu(), see.cpu())
    want = (ref.detach(), *torch.autograd.grad(ref, plain, do.double().cpu()))
    for name, a, b in zip(("out", "x", "wqkv", "wo", "wq", "wk"), got, want):
        off = float((a.double().cpu() - b).norm() / b.norm())
        assert off <= 12 * 2.0 ** -8, (name, off)
    # the same bits under checkpointing (the forward is run again) and with what is saved kept on the host meanwhile
    leaves = [t.clone().requires_grad_() for t in args]
    out = torch.utils.checkpoint.checkpoint(layer, *leaves, pos, freq, ranges, use_reentrant=False)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, do), got[1:]))
    leaves = [t.clone().requires_grad_() for t in args]
    with torch.autograd.graph.save_on_cpu():
        out = layer(*leaves, pos, freq, ranges)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, do), got[1:]))


def test_attention_gradients_against_differences(dev):
    """The gradients against central differences of the operator itself, in fp16 with steps that its inputs hold exactly.

    L = sum(out * do) in 64 bits over n = B Hq Sq D = 1536 rounded outputs below 4: each is off by 2^-11 * 4 at most and without a pattern,
    so (L+ - L-) / 2h by about sqrt(2 n) 2^-10 |do| / sqrt(3) / 2h = 0.13 at h = 1/8, and by h^2 / 6 of the third derivative along the way
    (1 / 384 of a value of the slope's size).  1 + 2 % of the slope is six times the first."""
    g = torch.Generator(device=dev).manual_seed(11)
    quarter = lambda *s: (torch.randn(*s, generator=g, device=dev).clamp(-3, 3) * 8).round().div(8).half()  # noqa: E731
    q, k, v, do = quarter(1, 2, 12, 64), quarter(1, 1, 12, 64), quarter(1, 1, 12, 64), quarter(1, 2, 12, 64)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.attention(*leaves, causal=True), leaves, do)
    loss = lambda *a: float((ops.attention(*a, causal=True).double() * do.double()).sum())  # noqa: E731
    h = 0.125
    for i, d in enumerate(grads):
        for _ in range(4):
            way = torch.randint(-1, 2, leaves[i].shape, generator=g, device=dev).half()
            way[torch.rand(way.shape, generator=g, device=dev) < 0.9] = 0
            up, down = ([*(t.detach() for t in leaves)] for _ in range(2))
            up[i], down[i] = up[i] + h * way, down[i] - h * way
            slope = (loss(*up) - loss(*down)) / (2 * h)
            assert abs(slope - float((d.double() * way.double()).sum())) <= 1 + 0.02 * abs(slope), i


def test_prefill_and_denoise_steps(dev):
    """A prefill fills the cache, denoise steps write their tokens behind it and read all of it; eagerly and as a graph that is replayed."""
    n, C = 16, 128
    x, wqkv, _, wq, wk = parameters(dev, 3)
    freq = wl.text_inv_freq(D).to(dev)
    cache = ops.quantized_kv_cache(B, HKV, C, D, dev)
    filled = torch.tensor([S, S - 20], dtype=torch.int32, device=dev)  # the second row is padded
    with torch.no_grad():
        q, k, v = project(x, wqkv, wq, wk, positions(dev), freq)
        out = ops.attention(q, k, v, key_lengths=torch.full_like(filled, S), causal=True)
        ops.kv_cache_write(k, v, *cache, torch.zeros_like(filled), lengths=filled)
        assert not cache[2][1, :, S - 20:].any() and not cache[0][1, :, S - 20:].float().any()
        # the cache in the place of k and v: the last query of every row sees the quantised keys of its row
        q1, k1, v1 = q[:1], *(c[:1, :, :S].double() * s[:1, :, :S, None].double() for c, s in zip(cache[:2], cache[2:]))
        check(ops.cached_attention(q1, *(c[:1].contiguous() for c in cache), key_lengths=filled[:1], causal=True),
              reference(q1, k1, v1, visible(1, S, S, dev, causal=True))["out"], "prompt over the cache")
        assert float((out[:1].double() - ops.cached_attention(q1, *(c[:1].contiguous() for c in cache), key_lengths=filled[:1], causal=True).double()).norm()
                     / out[:1].double().norm()) < 2.0 ** -4  # keys and values within half a step of e4m3

        action = torch.empty(B, n, H, dtype=torch.bfloat16, device=dev)
        pos = (filled.long()[None, :, None] + torch.arange(n, device=dev)).expand(3, B, n).contiguous()

        def step(own):
            q, k, v = project(action, wqkv, wq, wk, pos, freq)
            ops.kv_cache_write(k, v, *own, filled)
            return q, ops.cached_attention(q, *own, key_lengths=filled + n)

        g = torch.Generator(device=dev).manual_seed(4)
        mine = [c.clone() for c in cache]
        action.copy_(torch.randn(B, n, H, generator=g, device=dev))
        step(mine)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            made = step(mine)
        for turn in range(4):
            action.copy_(torch.randn(B, n, H, generator=g, device=dev))
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in made]
            other = [c.clone() for c in cache]
            q, want = step(other)
            assert torch.equal(got[0], q) and torch.equal(got[1], want), turn
            kk, vv = (c.double() * s.double()[..., None] for c, s in zip(other[:2], other[2:]))
            check(want, reference(q, kk, vv, visible(B, n, C, dev, lengths=filled + n))["out"], f"step {turn}")
            # the prompt's part of the cache is as it was, and so is what lies behind the step
            for b in range(B):
                a, e = int(filled[b]), int(filled[b]) + n
                for c, o in zip(cache, mine):
                    c, o = ((t.view(torch.uint8) if t.dim() == 4 else t) for t in (c, o))
                    assert torch.equal(c[b, :, :a], o[b, :, :a]) and torch.equal(c[b, :, e:], o[b, :, e:])


def test_two_graphs_on_two_streams(dev):
    """Captured training steps and generation steps, replayed at once on two streams: none shares a workspace with another."""
    freq, pos = wl.text_inv_freq(D).to(dev), positions(dev)
    ranges = ops.attention_key_ranges(types_of(dev))
    g = torch.Generator(device=dev).manual_seed(5)
    do = torch.randn(B, S, H, generator=g, device=dev).to(torch.bfloat16)
    one = torch.randn(B, HQ, 1, D, generator=g, device=dev).to(torch.bfloat16)
    long = torch.randn(B, HKV, 3000, D, generator=g, device=dev).to(torch.bfloat16)

    def run(args):
        leaves = [t.detach().requires_grad_() for t in args]
        out = layer(*leaves, pos, freq, ranges)
        return [out.detach(), *torch.autograd.grad(out, leaves, do), ops.attention(one, long, long)]

    sets = [parameters(dev, seed) for seed in (7, 8)]
    want = [[t.clone() for t in run(a)] for a in sets]
    torch.cuda.synchronize()
    graphs, made = [torch.cuda.CUDAGraph() for _ in sets], []
    for graph, a in zip(graphs, sets):
        with torch.cuda.graph(graph):
            made.append(run(a))
    streams = [torch.cuda.Stream() for _ in sets]
    for turn in range(5):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for m, w in zip(made, want):
            assert all(torch.equal(a, b) for a, b in zip(m, w)), turn
        run(sets[0])


@pytest.mark.parametrize("general", [False, True])
def test_capture_beside_an_eager_graph_of_the_same_leaves(dev, general):
    """A backward pass captured while an earlier graph of the leaves lives would have the default stream wait for the capturing one: the
    ops refuse it, and the capture goes through once that graph is gone."""
    g = torch.Generator(device=dev).manual_seed(6)
    order = (lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)) if general else (lambda t: t)  # (strides that the general path copies)
    q, k, v = (order(torch.randn(1, h, 20, D, generator=g, device=dev).to(torch.bfloat16)).requires_grad_() for h in (4, 2, 2))
    w = torch.ones(D, dtype=torch.bfloat16, device=dev, requires_grad=True)
    pos, freq = torch.arange(20, device=dev).expand(3, 1, 20).contiguous(), wl.text_inv_freq(D).to(dev)
    for op, leaves in ((lambda: ops.attention(q, k, v, causal=True), (q, k, v)),
                       (lambda: ops.qk_norm_rope_from_positions(q, k, w, w, pos, freq, SECTION)[0], (q, w))):
        alive = op()
        do = torch.ones_like(alive)
        want = torch.autograd.grad(op(), leaves, do)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="earlier graph of the same leaves"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                torch.autograd.grad(op(), leaves, do)
        torch.cuda.synchronize()
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            made = torch.autograd.grad(op(), leaves, do)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(made, want))


@pytest.mark.parametrize("mask_mode,fuse", [("causal", True), ("action_block", True), ("action_block", False)])
def test_prefill_harness(dev, mask_mode, fuse):
    """The harness on the library's attention, eagerly and replayed, against the plain forward: the bound of the harness's own test."""
    from wallx_mi355 import harness

    h = harness.PrefillHarness(n_layers=2, hidden=256, n_q=4, n_kv=2, head_dim=128, inter=(512, 256), vocab=151936, device=dev, seed=3, mask=mask_mode,
                               keep_dense=True, fuse=fuse, attention_native=True)
    row = wl.vla_row_tokens(n_images=1, image_tokens=16, lead_text=5, tail_text=9, n_action=8)
    ids = torch.tensor([row, row, row], dtype=torch.int64, device=dev)
    grid = torch.tensor([[1, 8, 8]] * 3, dtype=torch.int64, device=dev)
    types = ids == wl.ACTION_TOKEN_ID
    timer = harness.OpTimer()
    got = h.forward(ids, grid, types, timer)
    split = timer.report_ms()
    assert "attention" in split and "sdpa_torch" not in split and ("attention_ranges" in split) == (mask_mode == "action_block")
    ref = _ref_forward(h, ids, grid, types, mask_mode)
    assert float((got.float().cpu() - ref).abs().max()) <= 0.04 * float(ref.abs().max())
    if fuse:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            made = h.forward(ids, grid, types)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(made, got) and torch.equal(h.forward(ids, grid, types), got)
