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
