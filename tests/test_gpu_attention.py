"""Attention and its gradients against the formulas in 64 bits, under every kind of mask the key ranges can say.

Tolerances are bounds, not guesses.  With u half a step of the type (eps / 2) and |.| elementwise:
  O    u |O| (the result's rounding) + u P |V| (each probability's), and 2^-12 P |V| for fp32 scores, powers and sums (a score is
       off by at most D 2^-24 |q| |k| scale, below 2^-13 here);
  dV   the same of P^T dO;
  dS   u |dS|, P times the error of delta = sum dO O (O as rounded: |dO| tol(O)), and 2^-12 of |dS| + 2^-16 P |dO| |V| for fp32;
  dQ   u |dQ| + scale tol(dS) |K|, dK likewise with |Q|.
fp16 probabilities and slopes below 2^-14 lose up to 2^-25 each, and so does a result: fp16 numbers below 2^-14 are 2^-24 apart, so
that u |x| alone is less than half a step there."""

import math

import pytest
import torch

from wallx_mi355 import native
from wallx_mi355.fusions import ops

pytestmark = pytest.mark.gpu


def visible(B, Sq, Sk, dev, ranges=None, lengths=None, causal=False):
    j, i = torch.arange(Sk, device=dev), torch.arange(Sq, device=dev)[:, None]
    end = torch.full((B, 1, 1), Sk, device=dev) if lengths is None else lengths.clamp(0, Sk).view(B, 1, 1).long()
    see = (j < end).expand(B, Sq, Sk)
    if causal:
        see = see & (j <= end - Sq + i)
    if ranges is not None:
        see = see & (j >= ranges[..., :1]) & (j < ranges[..., 1:])
    return see[:, None]


def reference(q, k, v, see, scale=None, do=None):
    """{name: (value, tolerance)} in 64 bits."""
    u = torch.finfo(q.dtype).eps / 2
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    G, D = q.size(1) // k.size(1), q.size(3)
    scale = D ** -0.5 if scale is None else scale
    q, k, v = (t.double().contiguous() for t in (q, k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)))
    k, v = (torch.where(see.any(2)[..., None], t, 0.0) for t in (k, v))  # keys that no query sees
    T = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731
    s = (q @ T(k) * scale).masked_fill(~see, -math.inf)
    m = s.amax(-1, keepdim=True).clamp(min=-1e300)
    p = torch.exp(s - m)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    o = p @ v
    to = u * o.abs() + (u + 2.0 ** -12) * (p @ v.abs()) + tiny * (see.double() @ v.abs()) + tiny + 1e-30
    out = {"out": (o, to)}
    if do is not None:
        do = do.double().contiguous()
        seen = see.any(-1, keepdim=True)
        do, q = torch.where(seen, do, 0.0), torch.where(seen, q, 0.0)
        dp = do @ T(v)
        delta = (do * o).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        e = (u + 2.0 ** -12) * ds.abs() + p * ((do.abs() * to).sum(-1, keepdim=True) + 2.0 ** -16 * (do.abs() @ T(v.abs()))) + tiny * see
        dq, dk, dv = scale * (ds @ k), scale * (T(ds) @ q), T(p) @ do
        tq = u * dq.abs() + scale * (e @ k.abs())
        tk, tv = scale * (T(e) @ q.abs()), (u + 2.0 ** -12) * (T(p) @ do.abs()) + tiny * (T(see.double().expand_as(p)) @ do.abs())
        fold = lambda x: x.unflatten(1, (-1, G)).sum(2)  # noqa: E731
        dk, dv, tk, tv = fold(dk), fold(dv), fold(tk), fold(tv)
        out.update(dq=(dq, tq + tiny + 1e-30), dk=(dk, tk + u * dk.abs() + tiny + 1e-30), dv=(dv, tv + u * dv.abs() + tiny + 1e-30))
    return out


def check(got, want, what):
    value, tol = want
    assert got.shape == value.shape, what
    err = (got.double() - value).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off by up to {float((err / tol).nan_to_num(posinf=1e9).max()):.2f} tolerances"


def heads(B, S, H, D, dtype, g, dev):
    return torch.randn(B, S, H, D, generator=g, device=dev).to(dtype).transpose(1, 2)


def masks(kind, B, Sq, Sk, g, dev):
    i = torch.arange(Sq, device=dev)
    if kind == "full":
        return {}
    if kind == "causal":
        return dict(causal=True)
    if kind == "lengths":
        n = torch.randint(0, Sk + 1, (B,), generator=g, device=dev).to(torch.int32)
        n[0] = 0
        return dict(key_lengths=n, causal=True)
    if kind == "action":
        types = (i >= Sq - Sq // 3).expand(B, Sq)
        keep = i >= torch.randint(0, max(1, Sq // 2), (B, 1), generator=g, device=dev)
        return dict(key_ranges=ops.attention_key_ranges(types, keep))
    if kind == "packed":
        first = torch.rand(B, Sq, generator=g, device=dev) < 5.0 / Sq
        lo = torch.where(first, i, 0).cummax(1).values
        return dict(key_ranges=torch.stack((lo, (i + 1).expand(B, Sq)), -1).to(torch.int32))
    # any ranges at all: empty ones, reversed ones, ones beyond the keys
    return dict(key_ranges=torch.randint(-Sk // 2 - 1, Sk + Sk // 2 + 2, (B, Sq, 2), generator=g, device=dev).to(torch.int32),
                key_lengths=torch.randint(-3, Sk + 9, (B,), generator=g, device=dev).to(torch.int32))


def see_of(mask, B, Sq, Sk, dev):
    return visible(B, Sq, Sk, dev, mask.get("key_ranges"), mask.get("key_lengths"), mask.get("causal", False))


SIZES = [
    # B, Hq, Hkv, Sq, Sk, D
    (2, 4, 2, 1, 1, 128), (3, 8, 1, 1, 517, 128), (1, 2, 2, 3, 3, 64), (2, 6, 2, 33, 33, 80), (1, 3, 1, 65, 130, 64), (2, 8, 2, 100, 100, 128),
    (1, 7, 1, 129, 129, 80), (2, 2, 2, 200, 200, 128), (1, 16, 2, 257, 300, 128), (8, 4, 4, 70, 70, 64), (1, 1, 1, 640, 640, 128), (5, 14, 2, 17, 900, 128),
]


@pytest.mark.parametrize("mask", ["full", "causal", "lengths", "action", "packed", "any"])
@pytest.mark.parametrize("size", SIZES)
def test_forward_and_gradients(dev, size, mask):
    B, Hq, Hkv, Sq, Sk, D = size
    if mask in ("action", "packed"):
        Sk = Sq
    dtype = torch.bfloat16 if (Sq + D // 16 + len(mask)) % 2 else torch.float16
    g = torch.Generator(device=dev).manual_seed(Sq * 31 + Sk + D)
    q, k, v, do = heads(B, Sq, Hq, D, dtype, g, dev), heads(B, Sk, Hkv, D, dtype, g, dev), heads(B, Sk, Hkv, D, dtype, g, dev), heads(B, Sq, Hq, D, dtype, g, dev)
    kw = masks(mask, B, Sq, Sk, g, dev)
    want = reference(q, k, v, see_of(kw, B, Sq, Sk, dev), do=do)
    check(ops.attention(q, k, v, **kw), want["out"], "forward alone")
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.attention(*leaves, **kw)
    grads = torch.autograd.grad(out, leaves, do)
    for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads)):
        check(got, want[name], f"{name} {dtype}")
    again = torch.autograd.grad(ops.attention(*leaves, **kw), leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(grads, again)), "the gradients differ between two runs"


LONG = [(1, 16, 1, 8300, 150, 64), (1, 4, 1, 40, 9000, 128), (1, 6, 2, 2900, 2900, 80)]


@pytest.mark.parametrize("size,mask", [(s, m) for s in LONG for m in ("full", "causal", "any")] + [(LONG[2], "packed"), (LONG[2], "action")])
def test_gradients_of_long_axes(dev, size, mask):
    """More than 4096 blocks of 32 rows, more than 64 tiles of 64 keys, tiles whose rows are cut into many units."""
    B, Hq, Hkv, Sq, Sk, D = size
    g = torch.Generator(device=dev).manual_seed(Sq + D)
    dtype = torch.float16 if D == 80 else torch.bfloat16
    q, k, v, do = heads(B, Sq, Hq, D, dtype, g, dev), heads(B, Sk, Hkv, D, dtype, g, dev), heads(B, Sk, Hkv, D, dtype, g, dev), heads(B, Sq, Hq, D, dtype, g, dev)
    kw = masks(mask, B, Sq, Sk, g, dev)
    want = reference(q, k, v, see_of(kw, B, Sq, Sk, dev), do=do)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.attention(*leaves, **kw)
    for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, do))):
        check(got, want[name], f"{name} {dtype}")


@pytest.mark.parametrize("mask", ["full", "causal", "lengths", "any"])
def test_many_rows_over_many_keys(dev, mask):
    """Rows enough for the widest workgroups over more than 4096 keys, of which the last tile is not full."""
    B, Hq, Hkv, Sq, Sk, D = 4, 16, 2, 1030, 4111, 128
    g = torch.Generator(device=dev).manual_seed(len(mask))
    dtype = torch.float16 if mask == "any" else torch.bfloat16
    q, k, v, do = (heads(B, s, h, D, dtype, g, dev) for s, h in ((Sq, Hq), (Sk, Hkv), (Sk, Hkv), (Sq, Hq)))
    kw = masks(mask, B, Sq, Sk, g, dev)
    see = see_of(kw, B, Sq, Sk, dev)
    want = reference(q, k, v, see, do=do)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.attention(*leaves, **kw)
    for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, do))):
        check(got, want[name], f"{name} {dtype}")
    if mask == "lengths":  # what no query sees may hold anything
        unseen = ~see.any(2)[:, 0, :, None]
        k, v = (torch.where(unseen[:, None], bad, t) for bad, t in ((float("nan"), k), (float("inf"), v)))
        assert torch.equal(ops.attention(q, k, v, **kw), out)
    if mask == "causal":  # nor what only the last three see, for the others
        k, v = k.clone(), v.clone()
        k[:, :, -3:], v[:, :, -3:] = float("inf"), float("nan")
        got = ops.attention(q, k, v, **kw)
        check(got[:, :, :-3], tuple(x[:, :, :-3] for x in want["out"]), "rows before")
        assert torch.isnan(got[:, :, -3:]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("Hq,Hkv,Sq", [(16, 2, 912), (4, 4, 1000), (32, 1, 48), (8, 2, 6)])
def test_types_and_head_sizes(dev, dtype, D, Hq, Hkv, Sq):
    g = torch.Generator(device=dev).manual_seed(5)
    B, Sk = 2, 1000
    q, k, v, do = heads(B, Sq, Hq, D, dtype, g, dev), heads(B, Sk, Hkv, D, dtype, g, dev), heads(B, Sk, Hkv, D, dtype, g, dev), heads(B, Sq, Hq, D, dtype, g, dev)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.attention(*leaves, causal=True, scale=0.2)
    grads = torch.autograd.grad(out, leaves, do)
    want = reference(q, k, v, visible(B, Sq, Sk, dev, causal=True), 0.2, do)
    for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads)):
        check(got, want[name], name)


def test_scores_of_any_size(dev):
    """Scores far apart, in rising and falling order: the running maximum moves, and moves by little."""
    g = torch.Generator(device=dev).manual_seed(6)
    for factor in (0.0, 1e-3, 8.0, 60.0):
        q, k, v = (heads(1, n, 2, 128, torch.bfloat16, g, dev) for n in (150, 700, 700))
        rise = torch.linspace(-1, 1, 700, device=dev).view(1, 1, -1, 1)
        for sign in (1, -1):
            kk = (k.float() * 0.1 + sign * rise * factor * q.float().mean(2, keepdim=True).sign() / 12).to(torch.bfloat16)
            see = visible(1, 150, 700, dev)
            got = ops.attention(q, kk, v)
            value, tol = reference(q, kk, v, see)["out"]
            # (large scores: an error of D 2^-24 |q| |k| scale in the exponent)
            slack = 128 * 2.0 ** -24 * (q.double().abs() @ kk.double().abs().transpose(-1, -2).contiguous()).amax() * 128 ** -0.5
            check(got, (value, tol + 2 * slack * v.double().abs().amax()), f"factor {factor} {sign}")


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("Sq,Sk,Hq,Hkv", [(70, 70, 4, 2), (3, 300, 8, 1), (200, 200, 2, 2)])
def test_unseen_values_have_no_influence(dev, bad, Sq, Sk, Hq, Hkv):
    """Keys and values that some queries see and some do not, rows that see nothing and their gradients."""
    g = torch.Generator(device=dev).manual_seed(7)
    B, D, dtype = 2, 128, torch.bfloat16
    q, k, v, do = heads(B, Sq, Hq, D, dtype, g, dev), heads(B, Sk, Hkv, D, dtype, g, dev), heads(B, Sk, Hkv, D, dtype, g, dev), heads(B, Sq, Hq, D, dtype, g, dev)
    i = torch.arange(Sq, device=dev)
    cut = Sk - 20
    # queries of the last third see all keys from 5 on but the last 20; the first few see nothing; the others see 0..20
    lo = torch.where(i >= Sq - (Sq + 2) // 3, 5, 0)
    hi = torch.where(i >= Sq - (Sq + 2) // 3, cut, 20)
    hi = torch.where(i < Sq // 5, 0, hi)
    ranges = torch.stack((lo, hi), -1).to(torch.int32).expand(B, Sq, 2)
    see = visible(B, Sq, Sk, dev, ranges)
    want = reference(q, k, v, see, do=do)

    def run(q, k, v, do):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = ops.attention(*leaves, key_ranges=ranges)
        return (out.detach(), *torch.autograd.grad(out, leaves, do))

    k2, v2, q2, do2 = k.clone(), v.clone(), q.clone(), do.clone()
    k2[:, :, cut:], v2[:, :, cut:] = bad, bad                       # keys that nobody sees
    q2[:, :, :Sq // 5], do2[:, :, :Sq // 5] = bad, bad              # rows that see nothing
    for name, got in zip(("out", "dq", "dk", "dv"), run(q2, k2, v2, do2)):
        check(got, want[name], f"unseen {name}")
    # a value that only the last third sees: the other rows, and the gradients that do not depend on it, are as before
    v2[:, :, 30] = bad
    out, dq, dk, dv = run(q2, k2, v2, do2)
    near = slice(0, Sq - (Sq + 2) // 3)
    check(out[:, :, near], tuple(x[:, :, near] for x in want["out"]), "rows that do not see it")
    check(dq[:, :, near], tuple(x[:, :, near] for x in want["dq"]), "their gradients")
    assert not torch.isfinite(out[:, :, near.stop:]).any()
    check(dv, want["dv"], "dv does not depend on v")
    check(dk[:, :, :5], tuple(x[:, :, :5] for x in want["dk"]), "keys of the others alone")
    # a row whose gradient is not finite does not reach the keys that it does not see
    do3 = do.clone()
    do3[:, :, -1] = bad
    _, dq, dk, dv = run(q, k, v, do3)
    check(dk[:, :, :5], tuple(x[:, :, :5] for x in want["dk"]), "dk of unseen keys")
    check(dv[:, :, :5], tuple(x[:, :, :5] for x in want["dv"]), "dv of unseen keys")
    check(dq[:, :, :-1], tuple(x[:, :, :-1] for x in want["dq"]), "dq of other rows")
    assert not torch.isfinite(dv[:, :, 6:cut]).any()


def test_orders_in_memory(dev):
    g = torch.Generator(device=dev).manual_seed(8)
    B, Hq, Hkv, S, D = 2, 4, 2, 75, 128
    qkv = torch.randn(B, S, (Hq + 2 * Hkv) * D, generator=g, device=dev).to(torch.bfloat16)
    q, k, v = (t.unflatten(-1, (-1, D)).transpose(1, 2) for t in qkv.split([Hq * D, Hkv * D, Hkv * D], -1))
    do = heads(B, S, Hq, D, torch.bfloat16, g, dev)

    def run(q, k, v, do):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = ops.attention(*leaves, causal=True)
        return (out.detach(), *torch.autograd.grad(out, leaves, do))

    want = run(*(t.contiguous() for t in (q, k, v, do)))

    def odd(t):  # rows that are not on 16 bytes
        x = torch.empty(t.numel() + 3, dtype=t.dtype, device=dev)[3:].view(t.shape)
        return x.copy_(t)

    def last(t):  # the head's channels far apart
        return t.transpose(2, 3).contiguous().transpose(2, 3)

    for how in (lambda t: t, odd, last, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)):
        for a, b in zip(run(*(how(t) for t in (q, k, v, do))), want):
            assert torch.equal(a, b)
    one = k[:, :, :1].expand(B, Hkv, S, D)  # the same key everywhere, no memory of its own
    got = ops.attention(q, one, v[:1].expand(B, Hkv, S, D))
    check(got, reference(q, one, v[:1].expand(B, Hkv, S, D), visible(B, S, S, dev))["out"], "expanded")


@pytest.mark.parametrize("size", [(1, 40, 1, 20, 50, 64), (2, 64, 1, 9, 70, 128), (1, 130, 2, 7, 33, 80), (600, 1, 1, 3, 5, 64), (70000, 1, 1, 1, 1, 64)])
@pytest.mark.parametrize("mask", ["causal", "any"])
def test_groups_and_batches(dev, size, mask):
    """Groups of more than 32 heads, whole multiples of 32 and others, and batches of more rows than tiles."""
    B, Hq, Hkv, Sq, Sk, D = size
    g = torch.Generator(device=dev).manual_seed(Hq + B)
    q, k, v, do = (heads(B, s, h, D, torch.bfloat16, g, dev) for s, h in ((Sq, Hq), (Sk, Hkv), (Sk, Hkv), (Sq, Hq)))
    kw = masks(mask, B, Sq, Sk, g, dev)
    want = reference(q, k, v, see_of(kw, B, Sq, Sk, dev), do=do)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.attention(*leaves, **kw)
    for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, do))):
        check(got, want[name], name)


def test_broadcast_inputs(dev):
    """One prompt's keys and values for a batch, one query row for all: read through strides of zero, gradients summed by autograd."""
    g = torch.Generator(device=dev).manual_seed(12)
    B, Hq, Hkv, S, D = 3, 4, 2, 50, 128
    q, k, v = heads(1, 1, Hq, D, torch.bfloat16, g, dev), heads(1, S, Hkv, D, torch.bfloat16, g, dev), heads(1, S, 1, D, torch.bfloat16, g, dev)
    do = heads(B, S, Hq, D, torch.bfloat16, g, dev)
    wide = lambda q, k, v: (q.expand(B, Hq, S, D), k.expand(B, Hkv, S, D), v.expand(B, Hkv, S, D))  # noqa: E731
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.attention(*wide(*leaves), causal=True)
    grads = torch.autograd.grad(out, leaves, do)
    full = [t.contiguous().requires_grad_() for t in wide(q, k, v)]
    ref = ops.attention(*full, causal=True)
    assert torch.equal(out, ref)
    for a, b, leaf in zip(grads, torch.autograd.grad(ref, full, do), leaves):
        over = [d for d in range(4) if leaf.size(d) == 1 and b.size(d) > 1]
        assert torch.equal(a, b.sum(over, keepdim=True)) or float((a.double() - b.double().sum(over, keepdim=True)).abs().max()) <= 2.0 ** -8 * float(b.double().abs().sum(over).max())


@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("B,S,Hq,Hkv", [(5, 1, 12, 4), (1, 3, 64, 8), (2, 900, 3, 1), (9, 2000, 8, 2)])
def test_rows_of_one_key(dev, B, S, Hq, Hkv, D):
    """The probability of an only key does not move with its score: such rows give their queries and keys exactly nothing."""
    g = torch.Generator(device=dev).manual_seed(S)
    dtype = torch.float16 if S % 2 else torch.bfloat16
    q, k, v, do = (heads(B, S, h, D, dtype, g, dev) for h in (Hq, Hkv, Hkv, Hq))
    at = torch.arange(S, device=dev).expand(B, S)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    ranges = torch.stack((at, at + 1), -1).to(torch.int32)
    out = ops.attention(*leaves, ranges)
    dq, dk, dv = torch.autograd.grad(out, leaves, do)
    assert torch.equal(out, v.repeat_interleave(Hq // Hkv, 1)) and not dq.any() and not dk.any()
    check(dv, reference(q, k, v, visible(B, S, S, dev, ranges), do=do)["dv"], "dv")
    # the first row of a causal mask among others; and an only key that is not finite
    dq, dk, dv = torch.autograd.grad(ops.attention(*leaves, causal=True), leaves, do)
    assert not dq[:, :, 0].any()
    bad = v.clone()
    bad[:, :, 0] = float("nan")
    leaves[2] = bad.requires_grad_()
    dq, dk, _ = torch.autograd.grad(ops.attention(*leaves, ranges), leaves, do)
    assert torch.isnan(dq[:, :, 0]).all() and torch.isnan(dk[:, :, 0]).all() and not dq[:, :, 1:].any() and not dk[:, :, 1:].any()


def test_nothing_to_attend(dev):
    q = torch.randn(2, 4, 5, 64, device=dev, dtype=torch.bfloat16, requires_grad=True)
    e = torch.empty(2, 2, 0, 64, device=dev, dtype=torch.bfloat16, requires_grad=True)
    out = ops.attention(q, e, e)
    assert out.shape == q.shape and not out.any()
    (dq,) = torch.autograd.grad(out, q, torch.ones_like(out))
    assert not dq.any()
    k = torch.randn(2, 2, 9, 64, device=dev, dtype=torch.bfloat16, requires_grad=True)
    none = torch.empty(2, 4, 0, 64, device=dev, dtype=torch.bfloat16, requires_grad=True)
    out = ops.attention(none, k, k)
    assert out.shape == none.shape
    (dk,) = torch.autograd.grad(out, k, torch.ones_like(out))
    assert dk.shape == k.shape and not dk.any()
    assert ops.attention(q[:0], k[:0], k[:0]).shape == (0, 4, 5, 64)


def test_key_ranges_of_the_model(dev):
    B, S = 3, 40
    types = torch.zeros(B, S, dtype=torch.bool, device=dev)
    types[0, 30:38], types[1, 10:12] = True, True
    keep = torch.ones(B, S, dtype=torch.bool, device=dev)
    keep[0, :7], keep[1, 33:] = False, False
    see = torch.ones(S, S, dtype=torch.bool, device=dev).tril() | (types[:, :, None] & types[:, None, :])
    see = see & keep[:, None, :] & keep[:, :, None]
    r = ops.attention_key_ranges(types, keep)
    assert r.dtype == torch.int32
    assert torch.equal(visible(B, S, S, dev, r)[:, 0], see)
    assert torch.equal(visible(B, S, S, dev, ops.attention_key_ranges(types))[:, 0], torch.ones(S, S, dtype=torch.bool, device=dev).tril() | (types[:, :, None] & types[:, None, :]))
    types[2, 3], types[2, 9] = True, True
    native.set_checked(True)
    try:
        with pytest.raises(ValueError, match="one run"):
            ops.attention_key_ranges(types)
    finally:
        native.set_checked(False)


def test_long_offsets(dev):
    """A key and value tensor of more than 2^32 elements: positions whose byte offsets pass 32 bits."""
    B, H, D, S = 1, 1, 128, 40000
    stride = 120000  # elements between positions
    big = torch.zeros(S * stride + D, dtype=torch.bfloat16, device=dev)
    g = torch.Generator(device=dev).manual_seed(9)
    k, v = (big.as_strided((B, H, S, D), (0, 0, stride, 1), off) for off in (0, 60000))
    k.copy_(torch.randn(B, H, S, D, generator=g, device=dev))
    v.copy_(torch.randn(B, H, S, D, generator=g, device=dev))
    for Sq in (1, 150):
        q = heads(B, Sq, H, D, torch.bfloat16, g, dev)
        check(ops.attention(q, k, v, causal=True), reference(q, k, v, visible(B, Sq, S, dev, causal=True))["out"], "far keys")


def test_streams_and_graphs(dev):
    g = torch.Generator(device=dev).manual_seed(10)
    B, Hq, Hkv, S, D = 2, 8, 2, 130, 128
    q, k, v, do = (heads(B, S, h, D, torch.bfloat16, g, dev) for h in (Hq, Hkv, Hkv, Hq))
    one = heads(B, 1, Hq, D, torch.bfloat16, g, dev)

    def run():
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = ops.attention(*leaves, causal=True)
        return (out.detach(), *torch.autograd.grad(out, leaves, do), ops.attention(one, k, v))

    want = [t.clone() for t in run()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a, b in zip(run(), want):
            assert torch.equal(a, b)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = run()
    for turn in range(3):
        fresh = [torch.randn(t.shape, generator=g, device=dev).to(t.dtype) for t in (q, k, v, do, one)]
        for t, f in zip((q, k, v, do, one), fresh):
            t.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in made]
        for a, b in zip(got, run()):
            assert torch.equal(a, b), f"replay {turn}"
