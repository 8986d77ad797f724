"""The quantised key / value cache: what is written, bit for bit against fp32 division and rounding to nearest even, and attention over
it against the formulas in 64 bits on the values that the codes stand for (tolerances as in test_gpu_attention: the codes are
exact in both compute types)."""

import pytest
import torch

from test_gpu_attention import check, heads, reference, visible
from wallx_mi355.fusions import ops

pytestmark = pytest.mark.gpu


def quantise(x):
    most = torch.full((), 448.0, device=x.device)  # (divided by a Python number, torch multiplies by its reciprocal)
    scale = (x.float().abs().amax(-1) / most).clamp(min=2.0 ** -126)
    return (x.float() / scale[..., None]).to(torch.float8_e4m3fn), scale


def bits(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t.view(torch.int32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Hkv,S,C,D", [(1, 1, 1, 1, 128), (3, 2, 17, 40, 80), (2, 5, 100, 130, 64), (64, 2, 1, 50, 128), (2, 3, 33, 20, 128)])
def test_write(dev, B, Hkv, S, C, D, dtype):
    g = torch.Generator(device=dev).manual_seed(S)
    k, v = (heads(B, S, Hkv, D, dtype, g, dev) * torch.rand(B, 1, S, 1, generator=g, device=dev).mul(12).sub(6).exp().to(dtype) for _ in range(2))
    k, v = k.clone(), v.clone()
    k[0, 0, 0] = 0                                # a row of zeros
    v[0, -1, -1] = torch.finfo(dtype).tiny / 64 if dtype == torch.bfloat16 else 6e-8   # the smallest numbers
    v[-1, 0, 0, 3] = torch.finfo(dtype).max
    start = torch.randint(-5, C + 3, (B,), generator=g, device=dev).to(torch.int32)
    lengths = torch.randint(-1, S + 4, (B,), generator=g, device=dev).to(torch.int32)
    for n in (None, lengths):
        cache = list(ops.quantized_kv_cache(B, Hkv, C, D, dev))
        for t in cache:
            bits(t).copy_(torch.randint(0, 100, t.shape, generator=g, device=dev))
        want = [t.clone() for t in cache]
        for which, x in enumerate((k, v)):
            codes, scale = quantise(x)
            for b in range(B):
                for s in range(S if n is None else min(S, max(0, int(n[b])))):
                    at = int(start[b]) + s
                    if 0 <= at < C:
                        bits(want[which])[b, :, at] = bits(codes)[b, :, s]
                        want[2 + which][b, :, at] = scale[b, :, s]
        ops.kv_cache_write(k, v, *cache, start, lengths=n)
        for name, a, b in zip(("k", "v", "k scales", "v scales"), cache, want):
            assert torch.equal(bits(a), bits(b)), name


def test_write_every_number(dev):
    """All finite bf16 magnitudes beside a row's largest: every rounding, ties among them, and rows that are not finite."""
    x = torch.arange(0, 0x7f80, device=dev, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = torch.cat((x, -x, torch.zeros(-2 * x.numel() % 126, device=dev, dtype=torch.bfloat16))).view(-1, 126)
    for top in (2.0 ** -100, 1.0, 448.0, 3.0, 1e30):
        rows = torch.cat((x.clamp(-top, top), torch.full((x.size(0), 2), top, device=dev, dtype=torch.bfloat16)), 1)[None, None]
        cache = ops.quantized_kv_cache(1, 1, rows.size(2), 128, dev)
        ops.kv_cache_write(rows, rows, *cache, torch.zeros(1, dtype=torch.int32, device=dev))
        codes, scale = quantise(rows)
        assert torch.equal(cache[2], scale) and torch.equal(cache[0].float(), codes.float()) and torch.equal(bits(cache[0]), bits(cache[1]))
    bad = torch.ones(1, 1, 3, 128, dtype=torch.bfloat16, device=dev)
    bad[..., 1, 5], bad[..., 2, 127] = float("inf"), float("nan")
    cache = ops.quantized_kv_cache(1, 1, 4, 128, dev)
    ops.kv_cache_write(bad, bad, *cache, torch.ones(1, dtype=torch.int32, device=dev))
    back = cache[0].float() * cache[2][..., None]
    assert torch.equal(back[0, 0, 1], torch.ones(128, device=dev)) and torch.isnan(back[0, 0, 2:]).all() and not back[0, 0, 0].any()


def filled(B, Hkv, C, D, g, dev):
    (kc, ks), (vc, vs) = (quantise(torch.randn(B, Hkv, C, D, generator=g, device=dev) * 3) for _ in range(2))
    return kc, vc, ks, vs


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Hq,Hkv,Sq,C,D", [(2, 8, 1, 1, 1, 128), (3, 16, 2, 1, 1000, 128), (2, 16, 2, 32, 912, 128), (4, 4, 4, 5, 333, 64), (1, 7, 1, 50, 700, 80),
                                            (40, 16, 2, 32, 130, 128), (1, 2, 2, 300, 300, 64)])
def test_attention(dev, B, Hq, Hkv, Sq, C, D, dtype):
    g = torch.Generator(device=dev).manual_seed(C)
    kc, vc, ks, vs = filled(B, Hkv, C, D, g, dev)
    k, v = kc.double() * ks.double()[..., None], vc.double() * vs.double()[..., None]
    q = heads(B, Sq, Hq, D, dtype, g, dev) * 0.3
    lengths = torch.randint(0, C + 1, (B,), generator=g, device=dev).to(torch.int32)
    lengths[0] = C
    ranges = torch.stack((torch.randint(0, C, (B, Sq), generator=g, device=dev), torch.randint(0, C + 1, (B, Sq), generator=g, device=dev)), -1).to(torch.int32)
    for kw in (dict(), dict(key_lengths=lengths), dict(key_lengths=lengths, causal=True), dict(key_ranges=ranges, key_lengths=lengths)):
        want = reference(q, k, v, visible(B, Sq, C, dev, kw.get("key_ranges"), kw.get("key_lengths"), kw.get("causal", False)))["out"]
        check(ops.cached_attention(q, kc, vc, ks, vs, **kw), want, str(sorted(kw)))


@pytest.mark.parametrize("Hq,Hkv,Sq", [(8, 1, 1), (8, 2, 30), (2, 2, 150)])
def test_what_the_cache_holds_behind_the_length(dev, Hq, Hkv, Sq):
    g = torch.Generator(device=dev).manual_seed(2)
    B, C, D = 3, 400, 128
    kc, vc, ks, vs = filled(B, Hkv, C, D, g, dev)
    q = heads(B, Sq, Hq, D, torch.bfloat16, g, dev)
    lengths = torch.tensor([0, 200, 317], dtype=torch.int32, device=dev)
    want = [ops.cached_attention(q, kc, vc, ks, vs, key_lengths=lengths, causal=c) for c in (False, True)]
    assert not want[0][0].any()
    for b in range(B):
        n = int(lengths[b])
        bits(kc)[b, :, n:], bits(vc)[b, :, n:] = 0x7f, 0xff  # NaN
        ks[b, :, n:], vs[b, :, n:] = float("nan"), float("inf")
    for c in (False, True):
        assert torch.equal(ops.cached_attention(q, kc, vc, ks, vs, key_lengths=lengths, causal=c), want[c])
    # one within the length: the rows before it are as they were
    if Sq > 20:
        bits(vc)[2, :, 317 - 10] = 0x7f
        got = ops.cached_attention(q, kc, vc, ks, vs, key_lengths=lengths, causal=True)
        k, v = kc.double() * ks.double()[..., None], vc.double() * vs.double()[..., None]
        k[2, :, 317 - 10:], v[2, :, 317 - 10:] = 0, 0
        short = lengths.clone()
        value = reference(q, k.nan_to_num(), v.nan_to_num(), visible(B, Sq, C, dev, lengths=short, causal=True))["out"]
        check(got[2, :, :-10], tuple(x[2, :, :-10] for x in value), "rows before it")
        assert torch.isnan(got[2, :, -10:]).all()


def test_long_cache_and_graph(dev):
    """A cache whose byte offsets pass 32 bits, and its use in a replayed graph: a step written, then read."""
    B, Hkv, Hq, D, C = 1, 1, 8, 128, 34_000_000
    kc, vc = (torch.zeros(B, Hkv, C, D, dtype=torch.float8_e4m3fn, device=dev) for _ in range(2))
    ks, vs = (torch.ones(B, Hkv, C, dtype=torch.float32, device=dev) for _ in range(2))
    g = torch.Generator(device=dev).manual_seed(3)
    at = C - 700
    lo = torch.full((B, 1, 1), at, dtype=torch.int32, device=dev)
    ranges = torch.cat((lo, torch.full_like(lo, C)), -1)
    k, v, q = heads(B, 700, Hkv, D, torch.bfloat16, g, dev), heads(B, 700, Hkv, D, torch.bfloat16, g, dev), heads(B, 1, Hq, D, torch.bfloat16, g, dev)
    start = torch.full((B,), at, dtype=torch.int32, device=dev)

    def step():
        ops.kv_cache_write(k, v, kc, vc, ks, vs, start)
        return ops.cached_attention(q, kc, vc, ks, vs, key_ranges=ranges)

    def want():
        (a, sa), (b, sb) = quantise(k), quantise(v)
        return reference(q, a.double() * sa.double()[..., None], b.double() * sb.double()[..., None], visible(B, 1, 700, dev))["out"]

    check(step(), want(), "far positions")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(3):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        check(got, want(), f"replay {turn}")
        assert torch.equal(got, step())
