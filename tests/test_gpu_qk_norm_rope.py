"""The norm of q and k per head with M-RoPE against the formulas in 64 bits.  Tolerances: one rounding of the result, u |y| with u half
a step of the type, and fp32 arithmetic inside: a handful of operations each off by 2^-24 of |n cos| + |n' sin|, at most 2^-20 of
it (the head's sum of D squares included: D 2^-24 / 2 of it would be the worst order).  The gradients' fp32 errors likewise relative
to the sums of magnitudes; a weight's gradient sums T heads, each term off by 2^-20, in fp32 partial sums (2^-20 of the terms'
magnitudes more).  fp16 numbers below 2^-14 are 2^-24 apart: a result's rounding there is up to 2^-25, which u |y| falls short of."""

import pytest
import torch

from wallx_mi355 import native, workloads as wl
from wallx_mi355.fusions import ops

pytestmark = pytest.mark.gpu

SECTIONS = {64: [8, 8, 16], 128: [16, 24, 24], 256: [32, 48, 48]}
FP32 = 2.0 ** -20


def angles(pos, inv_freq, D, layout, section=None):
    s = section or SECTIONS[D]
    per = [0] * s[0] + [1] * s[1] + [2] * s[2]
    planes = per + per if layout == "hf" else [0] * (2 * s[0]) + [1] * (2 * s[1]) + [2] * (2 * s[2])
    a = torch.stack([pos[p].double() * inv_freq.double()[d % (D // 2)] for d, p in enumerate(planes)], -1)
    return a.cos()[:, None], a.sin()[:, None]


def turn(x):
    lo, hi = x.chunk(2, -1)
    return torch.cat((-hi, lo), -1)


def reference(x, w, cos, sin, eps, gy, dtype):
    u = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-38
    x, w = x.double(), w.double()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    n = x * r * w
    y = n * cos + turn(n) * sin
    ty = u * y.abs() + FP32 * ((n * cos).abs() + (turn(n) * sin).abs()) + tiny
    gy = gy.double()
    back = lambda g, s: g * cos - turn(g * s)  # noqa: E731  (rotate_half^T = -rotate_half)
    gn = back(gy, sin)
    big = (gy * cos).abs() + turn(gy * sin).abs()
    xh, gw = x * r, gn * w
    mean = (gw * xh).mean(-1, keepdim=True)
    dx = r * (gw - xh * mean)
    tx = u * dx.abs() + FP32 * r * (big * w.abs() + xh.abs() * (big * w.abs() * xh.abs()).mean(-1, keepdim=True)) + tiny
    dw = (gn * xh).sum((0, 1, 2))
    tw = u * dw.abs() + 2 * FP32 * (big * xh.abs()).sum((0, 1, 2)) + tiny
    return (y, ty), (dx, tx), (dw, tw)


def check(got, want, what):
    value, tol = want
    assert got.shape == value.shape, what
    err = (got.double() - value).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off by up to {float((err / tol).max()):.2f} tolerances"


def inputs(B, S, Hq, Hkv, D, dtype, far, dev, seed=1):
    g = torch.Generator(device=dev).manual_seed(seed)
    qkv = torch.randn(B, S, (Hq + 2 * Hkv) * D, generator=g, device=dev).to(dtype)
    q, k, _ = (t.unflatten(-1, (-1, D)).transpose(1, 2) for t in qkv.split([Hq * D, Hkv * D, Hkv * D], -1))
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g, device=dev)).to(dtype) for _ in range(2))
    pos = torch.randint(0, 2000, (3, B, S), generator=g, device=dev) + far
    gq, gk = (torch.randn(B, S, h, D, generator=g, device=dev).to(dtype).transpose(1, 2) for h in (Hq, Hkv))
    return q, k, wq, wk, pos, gq, gk


def run(op, q, k, wq, wk, gq, gk):
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    y = op(*leaves)
    return (*(t.detach() for t in y), *torch.autograd.grad(y, leaves, (gq, gk)))


def compare(got, q, k, wq, wk, cos, sin, eps, gq, gk, dtype):
    (yq, dq, dwq), (yk, dk, dwk) = reference(q, wq, cos, sin, eps, gq, dtype), reference(k, wk, cos, sin, eps, gk, dtype)
    for name, g, w in zip(("q", "k", "dq", "dk", "dwq", "dwk"), got, (yq, yk, dq, dk, dwq, dwk)):
        check(g, w, name)


@pytest.mark.parametrize("layout", ["hf", "csrc"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,S,Hq,Hkv,D,far", [(1, 1, 1, 1, 128, 0), (2, 37, 4, 2, 64, 900), (3, 211, 16, 2, 128, 30000), (1, 5, 14, 1, 256, 0), (2, 700, 2, 2, 64, 10 ** 6)])
def test_from_positions(dev, B, S, Hq, Hkv, D, far, dtype, layout):
    q, k, wq, wk, pos, gq, gk = inputs(B, S, Hq, Hkv, D, dtype, far, dev)
    freq = wl.text_inv_freq(D).to(dev)
    got = run(lambda *a: ops.qk_norm_rope_from_positions(*a, pos, freq, SECTIONS[D], eps=1e-5, layout=layout), q, k, wq, wk, gq, gk)
    compare(got, q, k, wq, wk, *angles(pos, freq, D, layout), 1e-5, gq, gk, dtype)
    assert got[0].is_contiguous() and got[1].is_contiguous()


@pytest.mark.parametrize("layout", ["hf", "csrc"])
@pytest.mark.parametrize("B,S,Hq,Hkv,D", [(64, 1, 16, 2, 128), (2, 37, 4, 2, 64), (3, 211, 16, 2, 128), (4, 3000, 7, 1, 128), (1, 3, 300, 0, 128), (1, 9, 0, 3, 64)])
def test_from_table(dev, B, S, Hq, Hkv, D, layout):
    dtype = torch.bfloat16
    q, k, wq, wk, pos, gq, gk = inputs(B, S, Hq, Hkv, D, dtype, 0, dev, 2)
    freq = wl.text_inv_freq(D).to(dev)
    table = ops.multimodal_rope_table(pos, freq, SECTIONS[D], layout)
    t = table.view(B, 1, S, -1)
    t = torch.cat((t, t), -1) if t.size(-1) == D // 2 else t
    cos, sin = (t << 16).view(torch.float32).double(), (t & -65536).view(torch.float32).double()
    got = run(lambda *a: ops.qk_norm_rope_from_table(*a, table, SECTIONS[D], layout=layout), q, k, wq, wk, gq, gk)
    compare(got, q, k, wq, wk, cos, sin, 1e-6, gq, gk, dtype)


@pytest.mark.parametrize("layout", ["hf", "csrc"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,section", [(64, [8, 12, 12]), (64, [1, 2, 29]), (128, [17, 20, 27]), (128, [64, 0, 0]), (32, [5, 6, 5])])
def test_sections_that_end_anywhere(dev, D, section, dtype, layout):
    B, S, Hq, Hkv = 2, 45, 6, 2
    q, k, wq, wk, pos, gq, gk = inputs(B, S, Hq, Hkv, D, dtype, 5000, dev, 4)
    freq = (10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float().to(dev)
    got = run(lambda *a: ops.qk_norm_rope_from_positions(*a, pos, freq, section, layout=layout), q, k, wq, wk, gq, gk)
    compare(got, q, k, wq, wk, *angles(pos, freq, D, layout, section), 1e-6, gq, gk, dtype)
    if dtype == torch.bfloat16:
        table = ops.multimodal_rope_table(pos, freq, section, layout)
        t = table.view(B, 1, S, -1)
        t = torch.cat((t, t), -1) if t.size(-1) == D // 2 else t
        cos, sin = (t << 16).view(torch.float32).double(), (t & -65536).view(torch.float32).double()
        got = run(lambda *a: ops.qk_norm_rope_from_table(*a, table, section, layout=layout), q, k, wq, wk, gq, gk)
        compare(got, q, k, wq, wk, cos, sin, 1e-6, gq, gk, dtype)


def test_against_differences(dev):
    """The gradients against central differences of the forward itself, in fp32: the step's own error is h^2 / 6 of the third
    derivative and 2^-24 |L| / h of the sums, both below 2e-2 here for a loss of a few hundred terms."""
    q, k, wq, wk, pos, gq, gk = inputs(1, 3, 2, 1, 64, torch.float32, 5, dev, 3)
    freq = wl.text_inv_freq(64).to(dev)
    op = lambda *a: ops.qk_norm_rope_from_positions(*a, pos, freq, SECTIONS[64])  # noqa: E731
    loss = lambda *a: sum((y.double() * g.double()).sum() for y, g in zip(op(*a), (gq, gk)))  # noqa: E731
    args = [q, k, wq, wk]
    grads = run(op, *args, gq, gk)[2:]
    g = torch.Generator(device=dev).manual_seed(4)
    for i, (a, d) in enumerate(zip(args, grads)):
        way = torch.randn(a.shape, generator=g, device=dev)
        h = 1e-2
        up, down = ([*args[:i], a + s * h * way, *args[i + 1:]] for s in (1, -1))
        slope = float((loss(*up) - loss(*down)) / (2 * h))
        assert abs(slope - float((d.double() * way.double()).sum())) <= 2e-2 * (1 + abs(slope)), i


def test_orders_in_memory_and_streams(dev):
    q, k, wq, wk, pos, gq, gk = inputs(2, 50, 4, 2, 128, torch.bfloat16, 0, dev, 5)
    freq = wl.text_inv_freq(128).to(dev)
    table = ops.multimodal_rope_table(pos, freq, SECTIONS[128])
    op = lambda *a: ops.qk_norm_rope_from_table(*a, table, SECTIONS[128])  # noqa: E731
    want = run(op, *(t.contiguous() for t in (q, k, wq, wk, gq, gk)))
    odd = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device=dev)[1:].view(t.shape).copy_(t)  # noqa: E731
    far = lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.dim() == 4 else t.repeat_interleave(2)[::2]  # noqa: E731
    for how in (lambda t: t, odd, far):
        for a, b in zip(run(op, *(how(t) for t in (q, k, wq, wk, gq, gk))), want):
            assert torch.equal(a, b)
    # a gradient that is one value for all
    ones = torch.ones((), dtype=torch.bfloat16, device=dev)
    got = run(op, q, k, wq, wk, ones.expand(gq.shape), ones.expand(gk.shape))
    for a, b in zip(got, run(op, q, k, wq, wk, torch.ones_like(gq), torch.ones_like(gk))):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(op, q, k, wq, wk, gq, gk)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = run(op, q, k, wq, wk, gq, gk)
    g = torch.Generator(device=dev).manual_seed(6)
    for _ in range(3):
        for t in (q, k, gq, gk):
            t.copy_(torch.randn(t.shape, generator=g, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in made]
        for a, b in zip(got, run(op, q, k, wq, wk, gq, gk)):
            assert torch.equal(a, b)


def test_rows_of_zeros_and_infinities(dev):
    q, k, wq, wk, pos, gq, gk = inputs(1, 8, 2, 2, 128, torch.bfloat16, 0, dev, 7)
    freq = wl.text_inv_freq(128).to(dev)
    q, k = q.clone(), k.clone()
    q[:, :, 3] = 0
    q[:, :, 5] = float("inf")
    got = run(lambda *a: ops.qk_norm_rope_from_positions(*a, pos, freq, SECTIONS[128]), q, k, wq, wk, gq, gk)
    assert not got[0][:, :, 3].any() and torch.isfinite(got[2][:, :, 3]).all()
    assert torch.isnan(got[0][:, :, 5]).all()
    assert torch.isfinite(got[0][:, :, [0, 1, 2, 3, 4, 6, 7]]).all() and torch.isfinite(got[3]).all()


def test_no_tokens(dev):
    D = 128
    q = torch.empty(2, 4, 0, D, dtype=torch.bfloat16, device=dev, requires_grad=True)
    w = torch.ones(D, dtype=torch.bfloat16, device=dev, requires_grad=True)
    table = torch.empty(0, D // 2, dtype=torch.int32, device=dev)
    y, z = ops.qk_norm_rope_from_table(q, q, w, w, table, SECTIONS[D])
    assert y.shape == q.shape
    (dw,) = torch.autograd.grad(y.sum() + z.sum(), w)
    assert not dw.any()
    assert native.mrope_table(torch.zeros(3, 1, 0, dtype=torch.int64, device=dev), wl.text_inv_freq(D).to(dev), SECTIONS[D]).shape[0] == 0
