"""Attention where the numbers are far from one: small and large values behind the cache's scales.

The bounds are those of test_gpu_attention, against the formulas in 64 bits, with what is said at each test; and, as errors that are
independent of one another add up to far less than their sum, a bound on the length of the error, 4 u of the result's with u half a
step of the type: the roundings that do not cancel (the probabilities', the result's) are each at most u of a term, the terms' signs are
random, and so the error's length is at most sqrt(2) u of the result's in the mean; numbers below 2^-14 in fp16 are 2^-24 apart, which
adds up to 2^-25 for each element."""

import pytest
import torch

from test_gpu_attention import check, heads, reference, visible
from test_gpu_kv_cache import quantise
from wallx_mi355 import native
from wallx_mi355.fusions import ops

pytestmark = pytest.mark.gpu
TINY = 2.0 ** -25


def near(got, value, what, slack=0.0):
    u = torch.finfo(got.dtype).eps / 2
    err, most = float((got.double() - value).norm()), 4 * u * float(value.norm()) + (TINY * value.numel() ** 0.5 if got.dtype == torch.float16 else 0.0) + slack
    assert err <= most, f"{what}: the error's length is {err / most:.2f} of what it may be"


CACHED = [  # B, Hq, Hkv, Sq, C, D: one query, some, many, split over the keys
    (2, 8, 1, 1, 900, 128), (2, 16, 2, 32, 912, 128), (1, 7, 1, 50, 700, 80), (80, 16, 2, 32, 300, 64), (4, 16, 2, 1, 12000, 128)]


def cached(q, k, v, **kw):
    """The op's result, and the reference's with its tolerance and one more 2^-25: an fp16 operand below 2^-14 is off by so much, under
    weights that sum to one."""
    (kc, ks), (vc, vs) = quantise(k), quantise(v)
    kd, vd = kc.double() * ks.double()[..., None], vc.double() * vs.double()[..., None]
    value, tol = reference(q, kd, vd, visible(q.size(0), q.size(2), k.size(2), q.device, kw.get("key_ranges"), kw.get("key_lengths"), kw.get("causal", False)))["out"]
    return ops.cached_attention(q, kc, vc, ks, vs, **kw), value, tol + (TINY if q.dtype == torch.float16 else 0.0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sigma", [1e-4, 1e-3, 1e-2, 1.0, 100.0])
@pytest.mark.parametrize("B,Hq,Hkv,Sq,C,D", CACHED)
def test_cached_values_of_any_size(dev, B, Hq, Hkv, Sq, C, D, sigma, dtype):
    g = torch.Generator(device=dev).manual_seed(C)
    q, k = heads(B, Sq, Hq, D, dtype, g, dev), torch.randn(B, Hkv, C, D, generator=g, device=dev)
    v = torch.randn(B, Hkv, C, D, generator=g, device=dev) * sigma
    lengths = torch.randint(C // 2, C + 1, (B,), generator=g, device=dev).to(torch.int32)
    got, value, tol = cached(q, k, v, key_lengths=lengths)
    check(got, (value, tol), "values")
    near(got, value, "values", TINY * value.numel() ** 0.5 if dtype == torch.float16 else 0.0)


@pytest.mark.parametrize("B,Hq,Hkv,Sq,C,D", CACHED)
def test_cached_scales_far_apart(dev, B, Hq, Hkv, Sq, C, D):
    """Neighbouring keys whose values differ by up to 2^20."""
    g = torch.Generator(device=dev).manual_seed(C + 1)
    q, k = heads(B, Sq, Hq, D, torch.float16, g, dev), torch.randn(B, Hkv, C, D, generator=g, device=dev)
    v = torch.randn(B, Hkv, C, D, generator=g, device=dev) * torch.exp2(torch.randint(-13, 8, (B, Hkv, C, 1), generator=g, device=dev))
    for kw in ({}, dict(causal=True)):
        got, value, tol = cached(q, k, v, **kw)
        check(got, (value, tol), str(kw))


@pytest.mark.parametrize("B,Hq,Hkv,Sq,C,D", CACHED)
def test_cached_scales_beyond_fp16(dev, B, Hq, Hkv, Sq, C, D):
    """Values that fp16 does not hold (a cache that bfloat16 wrote): unseen, or with a weight that brings their part back into its range;
    and small codes under large scales."""
    g = torch.Generator(device=dev).manual_seed(C + 2)
    q, k = heads(B, Sq, Hq, D, torch.float16, g, dev) * 0.1 + 1, torch.randn(B, Hkv, C, D, generator=g, device=dev) * 0.1
    v = torch.randn(B, Hkv, C, D, generator=g, device=dev)
    far = torch.arange(C, device=dev) % 7 == 3
    hi = C // 7 * 7 - 3  # (behind a key that is not far)
    k[:, :, far] -= 2.2  # D = 64: 2.2 * 8 below the others, 2^-25
    v[:, :, far] *= 2.0 ** 20
    got, value, tol = cached(q, k, v, key_lengths=torch.full((B,), hi, dtype=torch.int32, device=dev))
    assert torch.isfinite(got).all()
    check(got, (value, tol), "light")
    v[:, :, hi:] = 2.0 ** 60
    ranges = torch.tensor([0, hi], dtype=torch.int32, device=dev).expand(B, Sq, 2).clone()
    if Sq > 1:
        ranges[:, -1, 1], v[:, :, C - 1] = C, 0.0  # one row sees more, so that the others' tiles hold what they do not see
    got, value, _ = cached(q, k, v, key_ranges=ranges)
    rows = slice(0, Sq - 1 if Sq > 1 else 1)
    check(got[:, :, rows], (value[:, :, rows], tol[:, :, rows]), "unseen")
    for power in (8, 15, 24):
        codes = torch.randint(1, 3, (B, Hkv, C, D), generator=g, device=dev).to(torch.uint8).view(torch.float8_e4m3fn)  # 1 or 2 times 2^-9
        vs = torch.full((B, Hkv, C), 2.0 ** power, device=dev)
        kc, ks = quantise(k * torch.linspace(0.1, 3, C, device=dev)[:, None])  # (rising scores: the running maximum is behind)
        kd, vd = kc.double() * ks.double()[..., None], codes.double() * vs.double()[..., None]
        want = reference(q, kd, vd, visible(B, Sq, C, dev))["out"]
        check(ops.cached_attention(q, kc, codes, ks, vs), want, f"scale 2^{power}")


GRADIENTS = [  # B, Hq, Hkv, Sq, Sk, D, causal: rows in workgroups of 64 and of 128, long keys in units and as they are, an odd group
    (1, 2, 1, 4096, 4096, 128, True), (1, 4, 1, 70, 8192, 64, False), (2, 6, 2, 900, 900, 80, True), (40, 16, 2, 300, 300, 128, True)]


def gradients(q, k, v, do, causal):
    """{name: (value, tolerance)}: those of test_gpu_attention without what fp16 loses below 2^-14.  A probability enters its product 2^15 times as
    large and is off by 2^-25 / 2^15 below 2^-29; a slope by 2^-40 likewise, or, where the slopes of the rows beside it are so large
    that it is scaled by less, by 2^-34 of the largest of them."""
    see = visible(q.size(0), q.size(2), k.size(2), q.device, causal=causal)
    want = reference(q, k, v, see, do=do)
    u, G, scale = torch.finfo(q.dtype).eps / 2, q.size(1) // k.size(1), q.size(3) ** -0.5
    q, k, v, do = (t.double().contiguous() for t in (q, k.repeat_interleave(G, 1), v.repeat_interleave(G, 1), do))
    T = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731
    p = torch.softmax((q @ T(k) * scale).masked_fill(~see, -float("inf")), -1)
    o, most = want["out"]
    o_tol = u * o.abs() + (u + 2.0 ** -12) * (p @ v.abs()) + TINY + TINY * (see.double() @ v.abs())
    ds = p * (do @ T(v) - (do * o).sum(-1, keepdim=True))
    lost = (2.0 ** -40 + 2.0 ** -34 * ds.abs().amax((1, 2, 3), keepdim=True)) * see
    e = (u + 2.0 ** -12) * ds.abs() + p * ((do.abs() * o_tol).sum(-1, keepdim=True) + 2.0 ** -16 * (do.abs() @ T(v.abs()))) + lost
    fold = lambda x: x.unflatten(1, (-1, G)).sum(2)  # noqa: E731
    (dq, _), (dk, _), (dv, _) = want["dq"], want["dk"], want["dv"]
    return {"dq": (dq, u * dq.abs() + scale * (e @ k.abs()) + TINY), "dk": (dk, u * dk.abs() + scale * fold(T(e) @ q.abs()) + TINY),
            "dv": (dv, u * dv.abs() + fold((u + 2.0 ** -12) * (T(p) @ do.abs()) + 2.0 ** -40 * (T(see.double().expand_as(p)) @ do.abs())) + TINY)}


def held(got, value, tol):
    """65520 and more is infinity in fp16: a result that may be as large may be that, and counts as right here."""
    beyond = torch.isinf(got) & (got.sign() == value.sign()) & (value.abs() + tol >= 65520) & (got.dtype == torch.float16)
    return torch.where(beyond, 0, got), torch.where(beyond, 0, value), tol


def take_gradients(q, k, v, do, **kw):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    return torch.autograd.grad(ops.attention(*leaves, **kw), leaves, do)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("grad,value", [(1e-4, 1.0), (1e-3, 1.0), (1.0, 1.0), (1.0, 1e-3), (1e3, 30.0)])
@pytest.mark.parametrize("B,Hq,Hkv,Sq,Sk,D,causal", GRADIENTS)
def test_gradients_of_any_size(dev, B, Hq, Hkv, Sq, Sk, D, causal, grad, value, dtype):
    """Slopes far below fp16's normal numbers (a small gradient over many keys) and beyond its largest (the first rows of a causal mask
    under a large one)."""
    g = torch.Generator(device=dev).manual_seed(Sq + Sk)
    q, k, v, do = heads(B, Sq, Hq, D, dtype, g, dev), heads(B, Sk, Hkv, D, dtype, g, dev), heads(B, Sk, Hkv, D, dtype, g, dev) * value, heads(B, Sq, Hq, D, dtype, g, dev) * grad
    want = gradients(q, k, v, do, causal)
    for name, got in zip(("dq", "dk", "dv"), take_gradients(q, k, v, do, causal=causal)):
        got, value, tol = held(got, *want[name])
        check(got, (value, tol), name)
        near(got, value, name)


def test_gradients_far_apart(dev):
    """Packed sequences, one's gradients 2^24 times another's: blocks of rows and tiles of keys hold both, and each sequence's are its own."""
    g = torch.Generator(device=dev).manual_seed(3)
    Hq, Hkv, S, D, each = 8, 2, 1200, 128, 75
    q, k, v, do = (heads(1, S, h, D, torch.float16, g, dev) for h in (Hq, Hkv, Hkv, Hq))
    at = torch.arange(S, device=dev)
    do = do * torch.where(at // each % 2 == 0, 2.0 ** 13, 2.0 ** -11)[:, None].to(torch.float16)
    ranges = torch.stack((at // each * each, at + 1), -1).to(torch.int32)[None]
    got = take_gradients(q, k, v, do, key_ranges=ranges)
    for n in range(S // each):
        part = slice(n * each, (n + 1) * each)
        for name, a, (value, tol) in zip(("dq", "dk", "dv"), got, gradients(q[:, :, part], k[:, :, part], v[:, :, part], do[:, :, part], True).values()):
            a, value, tol = held(a[:, :, part], value, tol)
            check(a, (value, tol), f"{name} of sequence {n}")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sigma", [64.0, 1.0, 2.0 ** -6, 2.0 ** -9])
@pytest.mark.parametrize("B,Hq,Hkv,S,D", [(2, 4, 2, 64, 128), (40, 16, 2, 96, 64), (1, 3, 1, 100, 80)])
def test_rests_of_the_output(dev, B, Hq, Hkv, S, D, sigma, dtype):
    """delta = sum dO O is the difference of large numbers here: the values differ by a twentieth of their size, the keys by a tenth, so that dQ's
    error is that of delta, sqrt(D) |dO| times what O's rounding leaves (u / sqrt 3 of it), which the rests take to an eighth: their
    three bits.  Everything else is below a tenth of the error without them (a slope's rounding, u / sqrt 3 of P sigma sqrt(D) / 20 over S keys,
    is 1 / (20 sqrt(S)) of it), so that half is more than what may be left."""
    g = torch.Generator(device=dev).manual_seed(S)
    q, k, v, do = heads(B, S, Hq, D, dtype, g, dev) * 0.1, 1 + 0.1 * heads(B, S, Hkv, D, dtype, g, dev), sigma * (1 + 0.05 * heads(B, S, Hkv, D, dtype, g, dev)), heads(B, S, Hq, D, dtype, g, dev)
    want = reference(q, k, v, visible(B, S, S, dev), 1.0, do)["dq"][0]
    out, lse, rest = native.attention_fwd(q, k, v, scale=1.0, want_lse=True)
    errors = [float((native.attention_bwd(do, q, k, v, out, lse, r, scale=1.0)[0].double() - want).norm()) for r in (rest, None)]
    assert errors[0] < 0.5 * errors[1], f"{errors[0] / errors[1]:.3f} of the error without"
