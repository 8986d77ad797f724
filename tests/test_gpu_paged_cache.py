"""The paged key / value cache: its bookkeeping against lists of pages in Python, its write bit for bit, and attention over it against the
formulas in 64 bits on the values that the pages hold (tolerances as in test_gpu_attention)."""

import random

import pytest
import torch

from test_gpu_attention import check, reference
from test_gpu_kv_cache import bits, quantise
from wallx_mi355 import native
from wallx_mi355.fusions import ops

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


# ----------------------------------------------------------------------------- bookkeeping
def resized(lengths, wanted, table, stack, count, ps, width, max_tokens):
    """The definition, a page at a time: (lengths, count, starts, slots, positions), table and stack changed in place."""
    lengths, wanted = ([min(max(x, 0), width * ps) for x in v] for v in (lengths, wanted))
    pages = lambda n: -(-n // ps)  # noqa: E731
    held = stack[:max(0, min(count, len(stack)))]
    freed = [table[r][p] for r in range(len(lengths)) for p in range(pages(wanted[r]), pages(lengths[r]))]
    held += freed[: len(stack) - len(held)][::-1]
    new, starts, slots, positions = [], [0], [], []
    for r, (n, w) in enumerate(zip(lengths, wanted)):
        have = pages(n)
        while have < pages(w) and held:
            table[r][have] = held.pop()
            have += 1
        new.append(w if w <= n else min(w, have * ps))
        for i in range(n, new[-1]):
            slots.append(table[r][i // ps] * ps + i % ps if table[r][i // ps] >= 0 else -1)
            positions.append(i)
        starts.append(len(slots))
    stack[count: len(held)] = held[count:]
    tail = max(0, max_tokens - len(slots))
    return new, len(held), [min(x, max_tokens) for x in starts], (slots + [-1] * tail)[:max_tokens], (positions + [0] * tail)[:max_tokens]


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def compare_resize(dev, lengths, wanted, table, stack, count, ps, max_tokens):
    width = len(table[0]) if table else 4
    args = [ints(lengths, dev), ints(wanted, dev), ints(table, dev).view(len(table), width), ints(stack, dev), ints([count], dev)]
    before = [t.clone() for t in args]
    want = resized(lengths, wanted, table, stack, count, ps, width, max_tokens)
    for _ in range(2):  # (the same again: what it reads is not among what it writes)
        got = ops.paged_kv_resize(*args, ps, max_tokens)
        for name, a, b in zip(("lengths", "count", "starts", "slots", "positions"), got, (want[0], [want[1]], *want[2:])):
            assert a.flatten().tolist() == list(b), name
        assert args[2].tolist() == table and args[3].tolist() == stack
        assert all(torch.equal(a, b) for a, b in zip(args[:2] + args[4:], before[:2] + before[4:]))
    return got


@pytest.mark.parametrize("R,width,ps,pages,seed", [(1, 1, 1, 1, 0), (1, 5, 16, 3, 1), (7, 9, 16, 40, 2), (64, 12, 7, 400, 3), (255, 6, 32, 900, 4), (257, 5, 1, 700, 5),
                                                   (1000, 8, 16, 4000, 6), (4096, 3, 48, 9000, 7), (3, 700, 8, 1500, 8)])
def test_resize(dev, R, width, ps, pages, seed):
    rng = random.Random(seed)
    lengths, table = [0] * R, [[-1] * width for _ in range(R)]
    stack, count = list(range(pages)), pages
    rng.shuffle(stack)
    for step in range(4):
        kind = [rng.choice(["stay", "one", "some", "end", "any"]) for _ in range(R)]
        wanted = [{"stay": n, "one": n + 1, "some": n + rng.randint(0, 3 * ps), "end": 0, "any": rng.randint(-2, width * ps + 3)}[k] for k, n in zip(kind, lengths)]
        max_tokens = sum(max(0, w - n) for w, n in zip(wanted, lengths)) + rng.choice([0, 5])
        got = compare_resize(dev, lengths, wanted, table, stack, count, ps, max_tokens)
        lengths, count = got[0].tolist(), int(got[1])
        owned = [table[r][p] for r in range(R) for p in range(-(-lengths[r] // ps))] + stack[:count]
        assert sorted(owned) == list(range(pages)), "a page is lost, or owned twice"


def test_resize_edges(dev):
    compare_resize(dev, [], [], [], [2, 1, 0], 3, 16, 4)                                      # no requests
    compare_resize(dev, [5, 0], [5, 0], [[3], [-1]], [0, 1, 2, -1], 3, 8, 0)                  # nothing to do, no tokens
    compare_resize(dev, [0, 0, 0], [100, 100, 100], [[-1] * 8 for _ in range(3)], list(range(9)), 9, 16, 300)  # the second gets 32, the third nothing
    compare_resize(dev, [16, 0], [0, 16], [[4], [-1]], [-1] * 5, 0, 16, 16)                   # a freed page is taken at once
    compare_resize(dev, [16, 3], [32, 9], [[4, -1], [-1, -1]], [7, -1], 1, 16, 40)            # a page that is none: no slots
    compare_resize(dev, [8, 8, 8], [0, 0, 0], [[0], [1], [2]], [5, -1], 1, 8, 2)              # a stack that is too small loses the last
    compare_resize(dev, [0, 4], [3, 9], [[-1] * 3, [0, -1, -1]], [1, 2, 3, -1], 3, 4, 5)      # more tokens than max_tokens


def test_a_growth_taken_back_restores_the_stack(dev):
    lengths, table, free, count = ops.paged_kv_tables(5, 40, 120, dev)
    want = ints([33, 0, 7, 100, 16], dev)
    lengths, count, *_ = ops.paged_kv_resize(lengths, want, table, free, count, 8, 200)
    held = free[: int(count)].clone()
    more, less, *_ = ops.paged_kv_resize(lengths, lengths + ints([9, 1, 80, 0, 50], dev), table, free, count, 8, 200)
    back, again, starts, slots, _ = ops.paged_kv_resize(more, lengths, table, free, less, 8, 10)
    assert torch.equal(back, lengths) and torch.equal(again, count) and torch.equal(free[: int(count)], held)
    assert not starts.any() and bool((slots == -1).all())


@pytest.mark.parametrize("inference", [False, True])
@pytest.mark.parametrize("max_tokens", [0, 1, 37])
def test_resize_results_are_tensors_of_their_own(dev, max_tokens, inference):
    with torch.inference_mode(inference):
        lengths, table, free, count = ops.paged_kv_tables(3, 4, 12, dev)
        got = ops.paged_kv_resize(lengths, ints([1, 0, max(0, max_tokens - 1)], dev), table, free, count, 16, max_tokens)
        for x, (size, dtype) in zip(got, ((3, torch.int32), (1, torch.int32), (4, torch.int32), (max_tokens, torch.int32), (max_tokens, torch.int64))):
            assert x.shape == (size,) and x.dtype == dtype and x.is_contiguous() and x.data_ptr() % 16 == 0 and x.is_inference() == inference
        for i, x in enumerate(got):  # (whatever is done to one leaves the others)
            others = [(y, y.clone(), y._version if not inference else 0) for j, y in enumerate(got) if j != i]
            x.add_(1).fill_(-77)
            assert all(torch.equal(y, z) and (inference or y._version == v) for y, z, v in others)


def test_resize_checked(dev):
    lengths, table, free, count = ops.paged_kv_tables(2, 4, 8, dev)
    native.set_checked(True)
    try:
        with pytest.raises(ValueError, match="max_tokens"):
            ops.paged_kv_resize(lengths, ints([9, 3], dev), table, free, count, 4, 11)
        ops.paged_kv_resize(lengths, ints([9, 3], dev), table, free, count, 4, 12)
    finally:
        native.set_checked(False)


# ----------------------------------------------------------------------------- write
@pytest.mark.parametrize("same", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,S,Hkv,D,ps,pages", [(1, 1, 1, 64, 1, 1), (1, 37, 2, 128, 16, 5), (5, 9, 3, 80, 7, 20), (64, 1, 2, 128, 16, 70), (2, 300, 8, 80, 48, 14)])
def test_write(dev, B, S, Hkv, D, ps, pages, dtype, same):
    g = torch.Generator(device=dev).manual_seed(S)
    qkv = torch.randn(B, S, 2 * Hkv * D + 8, generator=g, device=dev).to(dtype)
    k, v = qkv[..., : Hkv * D].view(B, S, Hkv, D).transpose(1, 2), qkv[..., Hkv * D: 2 * Hkv * D].view(B, S, Hkv, D).transpose(1, 2)
    if same:
        v[0, 0, 0, :2] = torch.tensor([float("nan"), float("-inf")], dtype=dtype, device=dev)
    cache = list(ops.paged_kv_cache(pages, Hkv, ps, D, dev, *([dtype] if same else [])))
    for t in cache:
        if t is not None:
            t.view(torch.uint8).copy_(torch.randint(0, 100, t.view(torch.uint8).shape, generator=g, device=dev))
    slots = torch.randperm(pages * ps, generator=g, device=dev)[: B * S].to(torch.int32)
    slots = torch.cat((slots, slots.new_full((B * S - slots.numel(),), -1)))
    slots[torch.rand(B * S, generator=g, device=dev) < 0.2] = -1
    slots[-1] = pages * ps  # just outside
    slots[:1] = torch.where(slots[:1] >= 0, slots[:1], -2 ** 31)
    want = [None if t is None else t.clone() for t in cache]
    for i, x in enumerate((k, v)):
        x = x.transpose(1, 2).reshape(B * S, Hkv, D)
        codes, scale = (x, None) if same else quantise(x)
        for t, slot in enumerate(slots.tolist()):
            if 0 <= slot < pages * ps:
                want[i].view(torch.uint8)[slot // ps, :, slot % ps] = codes.view(torch.uint8)[t]
                if not same:
                    want[2 + i][slot // ps, :, slot % ps] = scale[t]
    version = cache[0]._version
    ops.paged_kv_write(k, v, *cache, slots if B % 2 else slots.view(B, S))
    assert cache[0]._version > version
    for a, b in zip(cache, want):
        assert (a is None and b is None) or torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# ----------------------------------------------------------------------------- attention
def pool(pages, Hkv, ps, D, dtype, e4m3, g, dev):
    out = []
    for _ in range(2):
        x = torch.randn(pages, Hkv, ps, D, generator=g, device=dev) * 3
        out.append(quantise(x) if e4m3 else (x.to(dtype), None))
    return [out[0][0], out[1][0], out[0][1], out[1][1]]


def tables(lengths, ps, pages, width, rng, dev):
    order = list(range(pages))
    rng.shuffle(order)
    rows = []
    for n in lengths:
        need = -(-n // ps)
        rows.append([order.pop() for _ in range(need)] + [rng.choice([-1, 2 ** 31 - 1, 0])] * (width - need))
    return ints(rows, dev).view(len(lengths), width)


def wanted(q, cache, table, lengths, starts, causal, scale=None, bad=None):
    """(value, tolerance) of every token, request by request; zeros for tokens of none."""
    B, Hq, S, D = q.shape
    pages, Hkv, ps, _ = cache[0].shape
    flat = q.transpose(1, 2).reshape(B * S, Hq, D)
    value, tol = (torch.zeros(B * S, Hq, D, device=q.device, dtype=torch.float64) for _ in range(2))
    for r, n in enumerate(lengths):
        n = min(max(n, 0), table.size(1) * ps)
        first, last = starts[r], starts[r + 1]
        if first >= last or n == 0:
            continue
        at = torch.arange(n, device=q.device)
        page = table[r].long()[at // ps]
        ok = (page >= 0) & (page < pages)
        kv = []
        for i in range(2):
            x = cache[i][page.clamp(0, pages - 1), :, at % ps].double()
            if cache[2] is not None:
                x = x * cache[2 + i][page.clamp(0, pages - 1), :, at % ps].double()[..., None]
            kv.append(x.transpose(0, 1)[None])
        i = torch.arange(last - first, device=q.device)[:, None]
        see = ok & (at <= n - (last - first) + i) if causal else ok.expand(last - first, n)
        part = flat[first:last].transpose(0, 1)[None]
        got, t = reference(part, *kv, see[None, None], scale)["out"]
        value[first:last], tol[first:last] = got[0].transpose(0, 1), t[0].transpose(0, 1)
    back = lambda x: x.view(B, S, Hq, D).transpose(1, 2)  # noqa: E731
    return back(value), back(tol)


def prefix(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


CASES = [
    # Hq, Hkv, D, ps, queries of each request, lengths, e4m3
    (1, 1, 128, 16, [1], [1], True),
    (16, 2, 128, 16, [1] * 5, [1, 15, 16, 17, 900], True),
    (16, 2, 128, 16, [1, 1, 1], [3000, 0, 5000], False),
    (8, 1, 128, 64, [5, 0, 3, 1, 4], [700, 50, 3, 64, 65], False),
    (7, 1, 80, 7, [3, 9, 1], [3, 1000, 222], True),
    (14, 2, 64, 32, [1, 129, 1, 40], [4000, 300, 1, 40], True),
    (4, 4, 64, 1, [33, 2], [100, 77], False),
    (6, 2, 80, 48, [65, 1], [65, 500], False),
    (16, 2, 128, 128, [300, 257, 0, 1], [300, 1500, 0, 2], True),
    (2, 2, 128, 256, [600], [2000], False),
    (24, 1, 64, 16, [1, 2, 3, 4, 5, 6, 7], [100, 200, 300, 400, 500, 600, 700], True),
    (3, 3, 80, 16, [1] * 100, [37 * i % 211 for i in range(100)], True),
    (64, 1, 128, 8, [1, 2], [333, 1111], False),
    (1, 1, 64, 16, [1, 1], [33000, 70], True),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(dev, case, dtype, causal):
    Hq, Hkv, D, ps, counts, lengths, e4m3 = CASES[case]
    rng, g = random.Random(case), torch.Generator(device=dev).manual_seed(case)
    width = max(1, max(-(-n // ps) for n in lengths)) + 1
    pages = sum(-(-n // ps) for n in lengths) + 3
    cache = pool(pages, Hkv, ps, D, dtype, e4m3, g, dev)
    table = tables(lengths, ps, pages, width, rng, dev)
    starts = prefix(counts)
    T = starts[-1] + 5  # padding behind the last request
    q = torch.randn(1, T, Hq * D + 16, generator=g, device=dev).to(dtype)[..., : Hq * D].view(1, T, Hq, D).transpose(1, 2)
    scale = None if case % 2 else 0.31 / D ** 0.5
    want = wanted(q, cache, table, lengths, starts, causal, scale)
    out = ops.paged_attention(q, *cache, table, ints(lengths, dev), ints(starts, dev), causal=causal, scale=scale)
    assert out.stride() == (T * Hq * D, D, Hq * D, 1) and not out._is_view()
    check(out, want, f"{dtype}")
    assert not out[0, :, starts[-1]:].any()
    again = ops.paged_attention(q, *cache, table, ints(lengths, dev), ints(starts, dev), causal=causal, scale=scale)
    assert torch.equal(out, again)


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("B,S,D", [(64, 1, 128), (5, 32, 128), (3, 7, 80), (2, 130, 64)])
def test_rows_are_requests(dev, B, S, D, e4m3):
    """Without starts; and with starts that cut [B, S] tokens elsewhere."""
    rng, g = random.Random(S), torch.Generator(device=dev).manual_seed(S)
    lengths = [rng.randint(0, 900) for _ in range(B)]
    cache = pool(B * 57 + 1, 2, 16, D, torch.bfloat16, e4m3, g, dev)
    table = tables(lengths, 16, B * 57 + 1, 57, rng, dev)
    q = torch.randn(B, S, 8, D, generator=g, device=dev).to(torch.bfloat16).transpose(1, 2)
    for causal in (True, False):
        out = ops.paged_attention(q, *cache, table, ints(lengths, dev), causal=causal)
        check(out, wanted(q, cache, table, lengths, prefix([S] * B), causal), "rows")
        if S > 1:
            starts = sorted(rng.randint(0, B * S) for _ in range(B + 1))
            out = ops.paged_attention(q, *cache, table, ints(lengths, dev), ints(starts, dev), causal=causal)
            check(out, wanted(q, cache, table, lengths, starts, causal), "starts")


@pytest.mark.parametrize("counts,lengths", [
    ([1] * 64, [800 + 7 * i % 113 for i in range(64)]),              # items of about one length: a like number of workgroups each
    ([1] * 300, [1 + 17 * i % 90 for i in range(300)]),              # more requests than a workgroup has threads
    ([0, 2, 0, 0] * 300, [5, 40, 0, 9] * 300),                       # most of them without queries
    ([1] * 40 + [70] + [0] * 30 + [3] * 5 + [150, 65], [200] * 40 + [300] + [10] * 30 + [2500, 1, 64, 63, 65] + [150, 1000]),  # tiles of both kinds
    ([33] * 20, [40 + 90 * i for i in range(20)]),                   # tiles of few rows alone, lengths far apart
    ([9, 1, 100], [5, 0, 60]),                                       # fewer keys than queries
    ([1], [20000]), ([2] * 3, [9000, 1, 4000]),
    # items of many rows, 768 to 2048 of them (of up to 64 requests 4096): a workgroup for each; of more, or more requests than 256, shares
    ([17] * 200, [20 + i for i in range(200)]), ([100] * 60, [100 + 3 * i for i in range(60)]), ([1, 250] * 30, [30, 260] * 30),
    ([80] * 250, [80 + i % 7 for i in range(250)]), ([17] * 300, [17 + i % 50 for i in range(300)]),
])
@pytest.mark.parametrize("e4m3", [True, False])
def test_schedules(dev, counts, lengths, e4m3):
    rng, g = random.Random(len(counts)), torch.Generator(device=dev).manual_seed(len(counts))
    ps, D, pages = 16, 64, sum(-(-n // 16) for n in lengths) + 2
    cache = pool(pages, 2, ps, D, torch.bfloat16, e4m3, g, dev)
    table = tables(lengths, ps, pages, -(-max(lengths) // ps), rng, dev)
    starts = prefix(counts)
    q = torch.randn(1, starts[-1], 16, D, generator=g, device=dev).to(torch.bfloat16).transpose(1, 2)
    for causal in (True, False):
        out = ops.paged_attention(q, *cache, table, ints(lengths, dev), ints(starts, dev), causal=causal)
        check(out, wanted(q, cache, table, lengths, starts, causal), "schedule")


def test_wide_tables(dev):
    """Tables that could hold 2^30 keys a request (measures in more than a key), few of which are there; tokens before the first request."""
    rng, g = random.Random(5), torch.Generator(device=dev).manual_seed(5)
    ps, width, lengths, counts = 65536, 16383, [70000, 131000, 3, 65537], [2, 40, 0, 1]
    cache = pool(8, 2, ps, 64, torch.bfloat16, True, g, dev)
    table = tables(lengths, ps, 8, 2, rng, dev)
    table = torch.cat((table, table.new_full((4, width - 2), -1)), 1)
    starts = [7 + x for x in prefix(counts)]
    q = torch.randn(1, starts[-1] + 2, 8, 64, generator=g, device=dev).to(torch.bfloat16).transpose(1, 2)
    for causal in (True, False):
        out = ops.paged_attention(q, *cache, table, ints(lengths, dev), ints(starts, dev), causal=causal)
        check(out, wanted(q, cache, table[:, :2], lengths, starts, causal), "wide")
        assert not out[0, :, :7].any() and not out[0, :, -2:].any()


def test_nothing_to_attend_to(dev):
    cache = ops.paged_kv_cache(3, 2, 16, 64, dev)
    q = torch.randn(1, 9, 4, 64, device=dev).to(torch.bfloat16).transpose(1, 2)
    none = torch.zeros(0, 5, dtype=torch.int32, device=dev)
    assert not ops.paged_attention(q, *cache, none, ints([], dev), ints([4], dev)).any()                                        # no requests
    assert not ops.paged_attention(q, *cache, ints([[0]] * 3, dev), ints([0, -5, 0], dev), ints([0, 4, 4, 9], dev)).any()     # no keys
    assert not ops.paged_attention(q, *cache, ints([[0]] * 3, dev), ints([9, 9, 9], dev), ints([4, 4, 4, 4], dev)).any()      # no queries
    assert not ops.paged_attention(q, *cache, torch.zeros(3, 0, dtype=torch.int32, device=dev), ints([9, 9, 9], dev), ints([0, 4, 4, 9], dev)).any()  # no pages to a request
    empty = ops.paged_kv_cache(0, 2, 16, 64, dev)
    assert not ops.paged_attention(q, *empty, ints([[0]], dev), ints([9], dev)).any()                                          # no pages at all
    assert ops.paged_attention(q[:, :, :0], *cache, none, ints([], dev), ints([0], dev)).shape == (1, 4, 0, 64)
    ops.paged_kv_write(q[:, :2], q[:, :2], *empty, torch.zeros(9, dtype=torch.int32, device=dev))


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("n", [1, 4, 70])
def test_pages_that_are_none(dev, n, e4m3):
    """Page numbers outside of the pool, lengths beyond the table, starts beyond the tokens: not seen, and nothing else read."""
    rng, g = random.Random(n), torch.Generator(device=dev).manual_seed(n)
    Hq, Hkv, D, ps = 8, 2, 128, 16
    lengths = [400, 130, 90, 10 ** 6, -4]
    cache = pool(120, Hkv, ps, D, torch.bfloat16, e4m3, g, dev)
    table = tables([400, 130, 96, 400, 0], ps, 120, 25, rng, dev)
    table[0, 3], table[0, 20], table[1, :9], table[2, 5] = -1, 120, 2 ** 31 - 1, -2 ** 31
    starts = prefix([n] * 5)
    q = torch.randn(1, starts[-1], Hq, D, generator=g, device=dev).to(torch.bfloat16).transpose(1, 2)
    for causal in (True, False):
        out = ops.paged_attention(q, *cache, table, ints(lengths, dev), ints(starts, dev), causal=causal)
        check(out, wanted(q, cache, table, lengths, starts, causal), "bad pages")
        odd = [starts[0], starts[1], starts[2], starts[3], 10 ** 9, 2 ** 31 - 1]
        clamped = [min(x, starts[-1]) for x in odd]
        out = ops.paged_attention(q, *cache, table, ints(lengths, dev), ints(odd, dev), causal=causal)
        check(out, wanted(q, cache, table, lengths, clamped, causal), "starts beyond the tokens")


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 5, 40, 200])
def test_what_is_not_seen_does_not_count(dev, n, dtype, e4m3):
    """NaN and infinities behind a request's length, in its later tokens and in other requests' pages; what a query sees of them counts."""
    rng, g = random.Random(n), torch.Generator(device=dev).manual_seed(n)
    Hq, Hkv, D, ps, lengths = 8, 2, 64, 16, [n + 250, n + 37]
    cache = pool(70, Hkv, ps, D, dtype, e4m3, g, dev)
    table = tables(lengths, ps, 70, 30, rng, dev)
    starts = prefix([n, n])
    q = torch.randn(1, 2 * n, Hq, D, generator=g, device=dev).to(dtype).transpose(1, 2)
    clean = ops.paged_attention(q, *cache, table, ints(lengths, dev), ints(starts, dev), causal=True)
    want = wanted(q, cache, table, lengths, starts, True)
    check(clean, want, "clean")
    owned = {(int(table[r, i // ps]), i % ps) for r in range(2) for i in range(lengths[r])}
    nan, inf = float("nan"), float("inf")
    bad = [None if t is None else t.clone() for t in cache]
    for p in range(70):
        for s in range(ps):
            if (p, s) not in owned:
                if e4m3:
                    for i in range(2):
                        bad[i].view(torch.uint8)[p, :, s] = 0x7f
                        bad[2 + i][p, :, s] = rng.choice([nan, inf, -inf])
                else:
                    for i in range(2):
                        bad[i][p, :, s] = rng.choice([nan, inf, -inf])
    out = ops.paged_attention(q, *bad, table, ints(lengths, dev), ints(starts, dev), causal=True)
    assert torch.equal(out, clean)
    # the last token's key and value: its own query's affair alone
    last = lengths[0] - 1
    p, s = int(table[0, last // ps]), last % ps
    for what in ("key", "value"):
        odd = [None if t is None else t.clone() for t in bad]
        i = 0 if what == "key" else 1
        if e4m3:
            odd[i].view(torch.uint8)[p, 0, s, 5] = 0x7f
        else:
            odd[i][p, 0, s, 5] = nan if what == "key" else -inf
        out = ops.paged_attention(q, *odd, table, ints(lengths, dev), ints(starts, dev), causal=True)
        mine = torch.zeros_like(clean, dtype=torch.bool)
        if what == "key":
            mine[0, :4, n - 1] = True  # (the four query heads of key / value head 0)
        else:
            mine[0, :4, n - 1, 5] = True
        # (a row that is made again rounds its probabilities anew: like the first one it is within u |O| + (u + 2^-12) P |V| of the exact result,
        # and the two within twice that of each other, which is more than some steps of O where values cancel)
        check(out.masked_fill(mine, 0), (want[0].masked_fill(mine, 0), want[1]), what)
        assert bool((torch.isnan(out[mine]) if what == "key" or e4m3 else torch.isinf(out[mine])).all()), what


def test_requests_that_claim_the_same_tokens_over_and_over(dev):
    """starts that descend 2300 times: more work than any that ascend can ask for, and none of it is done."""
    R, T, width, ps = 4600, 4096, 512, 16
    k, v, ks, vs = ops.paged_kv_cache(2, 1, ps, 64, dev)
    q = torch.ones(1, 1, T, 64, dtype=torch.bfloat16, device=dev)
    starts = ints([T * (r % 2) for r in range(R + 1)], dev)
    out = ops.paged_attention(q, k, v, ks, vs, torch.zeros(R, width, dtype=torch.int32, device=dev), ints([width * ps] * R, dev), starts)
    assert not out.any()


def test_large_and_small_values_in_fp16(dev):
    """Scales beyond fp16's range in both directions."""
    rng, g = random.Random(1), torch.Generator(device=dev).manual_seed(1)
    for n in (1, 50):
        for size in (1e-6, 1e-3, 6e4):
            lengths, starts = [300, 77], prefix([n, n])
            cache = pool(30, 2, 16, 128, torch.float16, True, g, dev)
            codes, scale = quantise((torch.rand(30, 2, 16, 128, generator=g, device=dev) * 2 - 1) * size)
            cache[1], cache[3] = codes, scale
            table = tables(lengths, 16, 30, 20, rng, dev)
            q = torch.randn(1, 2 * n, 8, 128, generator=g, device=dev).to(torch.float16).transpose(1, 2)
            out = ops.paged_attention(q, *cache, table, ints(lengths, dev), ints(starts, dev), causal=True)
            check(out, wanted(q, cache, table, lengths, starts, True), f"{n} {size}")


def test_steps_of_generation(dev):
    """The operators together as a server uses them: prompts, single tokens, drafts of which some are taken back, requests that end and join;
    the same attention as over each request's own keys and values in a row."""
    rng, g = random.Random(9), torch.Generator(device=dev).manual_seed(9)
    R, Hq, Hkv, D, ps, pages = 6, 8, 2, 128, 16, 90
    lengths, table, free, count = ops.paged_kv_tables(R, 24, pages, dev)
    cache = ops.paged_kv_cache(pages, Hkv, ps, D, dev)
    history = [[torch.zeros(0, Hkv, D, device=dev, dtype=torch.bfloat16)] * 2 for _ in range(R)]
    held = [0] * R
    for step in range(8):
        want = list(held)
        for r in range(R):
            want[r] = rng.choice([held[r] + 1, held[r] + rng.randint(1, 6), held[r] + 1, 0 if held[r] else rng.randint(1, 200), max(0, held[r] - 3)])
        added = sum(max(0, w - h) for w, h in zip(want, held))
        T = added + 4
        lengths, count, starts, slots, positions = ops.paged_kv_resize(lengths, ints(want, dev), table, free, count, ps, T)
        assert lengths.tolist() == want
        qkv = torch.randn(1, T, (Hq + 2 * Hkv) * D, generator=g, device=dev).to(torch.bfloat16)
        q, k, v = (x.view(1, T, -1, D).transpose(1, 2) for x in qkv.split([Hq * D, Hkv * D, Hkv * D], -1))
        ops.paged_kv_write(k, v, *cache, slots)
        out = ops.paged_attention(q, *cache, table, lengths, starts, causal=True)
        at = starts.tolist()
        assert at[-1] == added and positions[:added].tolist() == [i for h, w in zip(held, want) for i in range(h, w)]
        for r in range(R):
            n = at[r + 1] - at[r]
            history[r] = [torch.cat((x[: min(held[r], want[r])], new[0, :, at[r]: at[r + 1]].transpose(0, 1))) for x, new in zip(history[r], (k, v))]
            assert history[r][0].size(0) == want[r]
            if n == 0:
                continue
            one = ops.quantized_kv_cache(1, Hkv, want[r], D, dev)
            ops.kv_cache_write(*(x.transpose(0, 1)[None] for x in history[r]), *one, ints([0], dev))
            (codes_k, codes_v, sk, sv) = one
            i, j = torch.arange(n, device=dev)[:, None], torch.arange(want[r], device=dev)
            see = (j <= want[r] - n + i)[None, None]
            kk, vv = codes_k.double() * sk.double()[..., None], codes_v.double() * sv.double()[..., None]
            check(out[:, :, at[r]: at[r + 1]], reference(q[:, :, at[r]: at[r + 1]], kk, vv, see)["out"], f"step {step} request {r}")
        held = want


def test_steps_in_a_graph(dev):
    """A step captured once and replayed: tables, write and attention with the lengths taken over on the device, eager work in between."""
    g = torch.Generator(device=dev).manual_seed(3)
    R, Hq, Hkv, D, ps, pages = 5, 8, 2, 64, 16, 120
    state = list(ops.paged_kv_tables(R, 20, pages, dev))
    cache = ops.paged_kv_cache(pages, Hkv, ps, D, dev)
    wanted_ = torch.zeros(R, dtype=torch.int32, device=dev)
    qkv = torch.zeros(1, R + 3, (Hq + 2 * Hkv) * D, dtype=torch.bfloat16, device=dev)

    def step(state, cache):
        lengths, table, free, count = state
        new, left, starts, slots, _ = ops.paged_kv_resize(lengths, wanted_, table, free, count, ps, R + 3)
        q, k, v = (x.view(1, R + 3, -1, D).transpose(1, 2) for x in qkv.split([Hq * D, Hkv * D, Hkv * D], -1))
        ops.paged_kv_write(k, v, *cache, slots)
        out = ops.paged_attention(q, *cache, table, new, starts, causal=True)
        lengths.copy_(new)
        count.copy_(left)
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([t.clone() for t in state], [t.clone() for t in cache])
    torch.cuda.current_stream().wait_stream(side)
    eager, eager_cache = [t.clone() for t in state], [t.clone() for t in cache]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(state, cache)
    for i in range(40):
        qkv.copy_(torch.randn(qkv.shape, generator=g, device=dev))
        wanted_.copy_(torch.where(torch.rand(R, generator=g, device=dev) < 0.05, 0, eager[0] + 1).to(torch.int32))
        graph.replay()
        want = step(eager, eager_cache)
        assert torch.equal(captured, want), i
        for a, b in zip((*state, *cache), (*eager, *eager_cache)):
            assert torch.equal(a.view(torch.uint8) if a.dtype == F8 else a, b.view(torch.uint8) if b.dtype == F8 else b), i


def test_both_hosts_and_other_streams(dev, monkeypatch):
    from wallx_mi355 import _lib

    def everything():
        g = torch.Generator(device=dev).manual_seed(4)
        lengths, table, free, count = ops.paged_kv_tables(3, 6, 20, dev)
        made = ops.paged_kv_resize(lengths, ints([20, 1, 64], dev), table, free, count, 16, 90)
        k, v = (torch.randn(1, 90, 2, 64, generator=g, device=dev).to(torch.bfloat16).transpose(1, 2) for _ in range(2))
        q = torch.randn(1, 90, 6, 64, generator=g, device=dev).to(torch.bfloat16).transpose(1, 2)
        out = [*made, table, free]
        for dtype in (F8, torch.bfloat16):
            cache = ops.paged_kv_cache(20, 2, 16, 64, dev, dtype)
            ops.paged_kv_write(k, v, *cache, made[3])
            out += [t.view(torch.uint8) for t in cache if t is not None]
            out.append(ops.paged_attention(q, *cache, table, made[0], made[2], causal=True, scale=0.2))
        return out

    fast = everything()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = everything()
    torch.cuda.current_stream().wait_stream(stream)
    monkeypatch.setattr(_lib, "_host", _lib._NoHost)
    for i, (a, b, c) in enumerate(zip(fast, everything(), other)):
        assert torch.equal(a, b) and torch.equal(a, c) and a.stride() == b.stride(), i


def test_refused(dev):
    cache = ops.paged_kv_cache(4, 2, 16, 64, dev)
    plain = ops.paged_kv_cache(4, 2, 16, 64, dev, torch.bfloat16)
    table, lengths = ints([[0, 1], [2, 3]], dev), ints([5, 20], dev)
    x = torch.zeros(2, 2, 1, 64, dtype=torch.bfloat16, device=dev)
    ok = dict(q=x, cache=cache, table=table, lengths=lengths, starts=None)

    def attend(**kw):
        a = {**ok, **kw}
        return ops.paged_attention(a["q"], *a["cache"], a["table"], a["lengths"], a["starts"])

    attend()
    attend(cache=plain)
    for kw in (dict(q=x.float()), dict(q=x[0]), dict(q=x.half(), cache=plain), dict(cache=(*cache[:2], None, None)), dict(cache=(*cache[:3], None)), dict(cache=(*plain[:2], *cache[2:])),
               dict(table=table.long()), dict(table=table[:1]), dict(lengths=lengths.long()), dict(lengths=lengths[:1]), dict(starts=ints([0, 1], dev)),
               dict(q=torch.zeros(2, 3, 1, 64, dtype=torch.bfloat16, device=dev)), dict(q=torch.zeros(2, 2, 1, 128, dtype=torch.bfloat16, device=dev)),
               dict(q=torch.zeros(3, 2, 1, 64, dtype=torch.bfloat16, device=dev)), dict(q=x.detach().clone().requires_grad_()), dict(lengths=lengths.cpu()),
               dict(cache=tuple(t.transpose(1, 2) for t in cache))):
        with pytest.raises(RuntimeError):
            attend(**kw)
    slots = ints([3, 40], dev)
    ops.paged_kv_write(x, x, *cache, slots)
    for args in ((x, x[:1], *cache, slots), (x, x, *cache, slots.long()), (x, x, *cache, slots[:1]), (x.float(), x.float(), *cache, slots), (x, x, *plain[:2], *cache[2:], slots),
                 (x.half(), x.half(), *plain, slots), (x[:, :1], x[:, :1], *cache, slots), (x.detach().clone().requires_grad_(), x, *cache, slots), (x, x, *cache, slots.cpu())):
        with pytest.raises(RuntimeError):
            ops.paged_kv_write(*args)
    state = ops.paged_kv_tables(2, 2, 4, dev)
    args = (state[0], lengths, *state[1:], 16, 30)
    ops.paged_kv_resize(*args)
    for at, wrong in ((1, lengths.long()), (1, lengths[:1]), (2, state[1].t()), (2, state[1].long()), (3, state[2].long()), (4, ints([1, 1], dev)), (5, 0), (5, -16), (6, -1),
                      (1, lengths.cpu()), (0, lengths.cpu())):
        with pytest.raises(RuntimeError):
            ops.paged_kv_resize(*args[:at], wrong, *args[at + 1:])
