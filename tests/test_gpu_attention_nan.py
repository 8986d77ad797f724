"""Numbers that are not finite: where NaN has to be, where it must not be, and that a step that overflowed takes no longer than another.

A sum is NaN exactly where a seen term is: with P_i NaN where query i, or a key that it sees, holds one,
  out[i, c]   P_i, or a seen v[j, c];
  dq[i, :]    P_i, or delta_i = sum dO O, which is NaN with any of row i's dO and out;
  dk[j, :]    any such row that sees j;
  dv[j, c]    P_i of a row that sees j, or its dO[i, c].
Everything else is what it is with the NaN taken as zeros: terms that are not there."""

import pytest
import torch

from test_gpu_attention import check, heads, masks, reference, see_of
from wallx_mi355.fusions import ops

pytestmark = pytest.mark.gpu
NAN = float("nan")


def expected(q, k, v, do, see):
    """{name: bool, where NaN has to be} over all heads of the queries, and for dk and dv of the keys."""
    G = q.size(1) // k.size(1)
    n = lambda t: torch.isnan(t)  # noqa: E731
    wide = lambda t: t.repeat_interleave(G, 1)  # noqa: E731
    see = see.expand(q.size(0), q.size(1), q.size(2), k.size(2)).double()
    some = see.any(-1, keepdim=True)
    p = some & (n(q).any(-1, keepdim=True) | (see @ wide(n(k)).any(-1, keepdim=True).double() > 0))
    out = p | (see @ wide(n(v)).double() > 0)
    row = p | (some & (n(do) | out).any(-1, keepdim=True))
    T = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731
    fold = lambda x: x.unflatten(1, (-1, G)).any(2)  # noqa: E731
    dk = fold(T(see) @ row.double() > 0)
    dv = fold(T(see) @ (p | n(do)).double() > 0)
    return {"out": out, "dq": row.expand_as(q), "dk": dk.expand_as(k), "dv": dv}


def put(where, q, k, v, do):
    """The tensors with NaN in the places that `where` names."""
    q, k, v, do = (t.clone() for t in (q, k, v, do))
    S, Sk = q.size(2), k.size(2)
    if where == "a token":  # as a layer's hidden state leaves it
        q[:, :, S // 3], k[:, :, Sk // 3], v[:, :, Sk // 3] = NAN, NAN, NAN
    elif where == "a query":
        q[0, 0, S // 2, 3] = NAN
    elif where == "a key":
        k[:, -1, Sk - Sk // 4, 5] = NAN
    elif where == "a value's channel":
        v[:, :, Sk // 2, 7] = NAN
    elif where == "values":
        v[:, :, Sk // 5:Sk // 5 + 3] = NAN
        v[:, 0, -2, 11] = NAN
    elif where == "all gradients":
        do[:] = NAN
    elif where == "a row's gradient":
        do[:, :, S - S // 3] = NAN
    else:  # channels of some gradients
        do[:, :, S // 2, 9], do[:, 1, S // 4, 60] = NAN, NAN
    return q, k, v, do


PLACES = ["a token", "a query", "a key", "a value's channel", "values", "all gradients", "a row's gradient", "gradients' channels"]


@pytest.mark.parametrize("where", PLACES)
@pytest.mark.parametrize("mask", ["full", "causal", "lengths", "packed", "any"])
@pytest.mark.parametrize("B,Hq,Hkv,Sq,Sk,D", [(2, 4, 2, 130, 130, 128), (1, 3, 1, 333, 333, 80), (9, 16, 2, 500, 500, 64), (2, 8, 2, 4, 3000, 128), (1, 16, 1, 4200, 4200, 128)])
def test_nan_is_where_it_has_to_be(dev, B, Hq, Hkv, Sq, Sk, D, mask, where):
    if Sq > 1000 and (mask not in ("causal", "packed") or where not in ("values", "a token", "all gradients")):
        pytest.skip("the long rows: two masks, three places")
    if mask == "packed" and Sq != Sk:
        pytest.skip("packed sequences are their own keys")
    g = torch.Generator(device=dev).manual_seed(Sq + D)
    dtype = torch.float16 if (D + len(mask)) % 3 else torch.bfloat16
    clean = [heads(B, s, h, D, dtype, g, dev) for s, h in ((Sq, Hq), (Sk, Hkv), (Sk, Hkv), (Sq, Hq))]
    kw = masks(mask, B, Sq, Sk, g, dev)
    see = see_of(kw, B, Sq, Sk, dev)
    bad = put(where, *clean)
    nan = expected(*bad, see)
    q, k, v, do = (t.nan_to_num(nan=0.0) for t in bad)
    want = reference(q, k, v, see, do=do)
    leaves = [t.detach().requires_grad_() for t in bad[:3]]
    out = ops.attention(*leaves, **kw)
    for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, bad[3]))):
        assert torch.equal(torch.isnan(got), nan[name]), f"{name}: {int((torch.isnan(got) != nan[name]).sum())} of {got.numel()}"
        value, tol = want[name]
        check(torch.where(nan[name], 0, got), (torch.where(nan[name], 0, value), tol), name)


@pytest.mark.parametrize("mask", ["causal", "lengths", "any"])
@pytest.mark.parametrize("B,Hq,Hkv,Sq,C,D", [(2, 8, 2, 1, 3000, 128), (2, 16, 2, 32, 912, 128), (1, 7, 1, 50, 700, 80), (40, 16, 2, 70, 300, 64)])
def test_nan_in_the_cache(dev, B, Hq, Hkv, Sq, C, D, mask):
    """A channel's code, a value's scale, a key's scale."""
    from test_gpu_kv_cache import bits, quantise

    g = torch.Generator(device=dev).manual_seed(C + D)
    for dtype in (torch.bfloat16, torch.float16):
        q = heads(B, Sq, Hq, D, dtype, g, dev)
        kw = masks(mask, B, Sq, C, g, dev)
        see = see_of(kw, B, Sq, C, dev)
        for which in range(3):
            (kc, ks), (vc, vs) = (quantise(torch.randn(B, Hkv, C, D, generator=g, device=dev)) for _ in range(2))
            if which == 0:
                bits(vc)[:, :, C // 3, 5], bits(vc)[:, 0, C - 5, 17] = 0x7f, 0xff
            elif which == 1:
                vs[:, :, C // 2] = NAN
            else:
                ks[:, 0, C - C // 3] = NAN
            k, v = kc.double() * ks.double()[..., None], vc.double() * vs.double()[..., None]
            nan = expected(q, k, v, q, see)["out"]
            value, tol = reference(q, k.nan_to_num(nan=0.0), v.nan_to_num(nan=0.0), see)["out"]
            got = ops.cached_attention(q, kc, vc, ks, vs, **kw)
            assert torch.equal(torch.isnan(got), nan), which
            check(torch.where(nan, 0, got), (torch.where(nan, 0, value), tol), str(which))


def timed(f):
    f()
    best = float("inf")
    for _ in range(3):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda.synchronize()
        a.record()
        f()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


@pytest.mark.parametrize("where", PLACES[:1] + PLACES[4:])
def test_a_step_that_overflowed_takes_no_longer(dev, where):
    """4 rows of 912 tokens with their gradients.  (What is not finite makes the kernels look at it again, which takes the time of some passes;
    in plain loops over every row it would be up to a hundred.)"""
    g = torch.Generator(device=dev).manual_seed(1)
    clean = [heads(4, 912, h, 128, torch.float16, g, dev) for h in (16, 2, 2, 16)]

    def step(q, k, v, do):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        return lambda: torch.autograd.grad(ops.attention(*leaves, causal=True), leaves, do)

    fine, bad = timed(step(*clean)), timed(step(*put(where, *clean)))
    assert bad < 10 * fine, f"{bad:.2f} ms, {fine:.2f} without"
