"""The paged cache at the edges of what its calls allow: buffers with room for many more tokens than a step has, against the formulas in 64 bits
(as in test_gpu_paged_cache)."""

import random

import pytest
import torch

from test_gpu_attention import check
from test_gpu_paged_cache import ints, pool, prefix, tables, wanted
from wallx_mi355 import _lib
from wallx_mi355.fusions import ops

pytestmark = pytest.mark.gpu


def guarded(q, cache, table, lengths, starts, causal):
    """The call in a workspace of just its size and with a result of its own, both between other memory, which stays as it is."""
    _, Hq, T, D = q.shape
    pages, Hkv, ps, _ = cache[0].shape
    guard, n, size = 64 << 20, _lib.load().wx_paged_attention_workspace_bytes(T, Hq, Hkv, D), T * Hq * D * 2
    work, out = (torch.full((x + 2 * guard,), 0x5A, dtype=torch.uint8, device=q.device) for x in (n, size))
    k_pages, v_pages, k_scale, v_scale = (None if t is None else t.data_ptr() for t in cache)
    _lib.call("wx_paged_attention", q.data_ptr(), k_pages, v_pages, k_scale, v_scale, out.data_ptr() + guard, table.data_ptr(), lengths.data_ptr(), starts.data_ptr(), int(causal), 1, Hq,
              Hkv, T, lengths.numel(), table.size(1), pages, ps, D, _lib.i64x3((0, q.stride(1), q.stride(2))), D ** -0.5, _lib.WX_BF16, work.data_ptr() + guard, n,
              torch.cuda.current_stream().cuda_stream)
    for buffer, x in ((work, n), (out, size)):
        assert bool((buffer[:guard] == 0x5A).all()) and bool((buffer[guard + x:] == 0x5A).all())
    return out[guard: guard + size].view(torch.bfloat16).view(1, T, Hq, D).transpose(1, 2)


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("counts,lengths,T,Hq,Hkv,D,causal", [
    ([1] * 16, [912] * 16, 16 * 912, 16, 2, 128, True),                                  # a token each, in equal parts
    ([1] * 64, [800 + 7 * i % 113 for i in range(64)], 8192, 16, 2, 128, True),
    ([3, 5, 1, 0] * 8, [700 + i for i in range(32)], 16 * 912, 16, 2, 128, True),        # drafts
    ([32] * 16, [860 + i for i in range(16)], 16 * 912, 16, 2, 128, False),              # a denoise step's
    ([1] * 8, [20000 + 700 * i for i in range(8)], 8192, 16, 2, 64, True),               # long contexts
    ([1] * 63 + [600], [400] * 63 + [1700], 16384, 16, 2, 64, True),                     # a chunk among them: both kinds of items
    ([1] * 100, [1 + 31 * i % 300 for i in range(100)], 9000, 16, 4, 80, True),          # more requests than a wavefront has lanes
    ([1] * 32, [500] * 32, 1024, 64, 8, 128, True),
])
def test_room_for_more_tokens(dev, counts, lengths, T, Hq, Hkv, D, causal, e4m3):
    """The launch is as wide as the buffer's items could be; nothing is done twice, or outside of the workspace."""
    rng, g = random.Random(T), torch.Generator(device=dev).manual_seed(T)
    ps, pages = 16, sum(-(-n // 16) for n in lengths) + 2
    cache = pool(pages, Hkv, ps, D, torch.bfloat16, e4m3, g, dev)
    table = tables(lengths, ps, pages, -(-max(lengths) // ps), rng, dev)
    starts = prefix(counts)
    q = torch.randn(1, T, Hq, D, generator=g, device=dev).to(torch.bfloat16).transpose(1, 2)
    want = wanted(q, cache, table, lengths, starts, causal)
    out = ops.paged_attention(q, *cache, table, ints(lengths, dev), ints(starts, dev), causal=causal)
    check(out, want, "room")
    assert not out[0, :, starts[-1]:].any()
    exact = ops.paged_attention(q[:, :, : starts[-1]], *cache, table, ints(lengths, dev), ints(starts, dev), causal=causal)
    check(exact, [x[:, :, : starts[-1]] for x in want], "no room")
    assert torch.equal(guarded(q, cache, table, ints(lengths, dev), ints(starts, dev), causal), out)


def test_a_captured_step_with_room_for_prompts(dev):
    """A step captured with max_tokens of sixteen prompts, replayed by prompts, by single tokens, by drafts and by nothing at all."""
    g, rng = torch.Generator(device=dev).manual_seed(8), random.Random(8)
    R, Hq, Hkv, D, ps, pages, T = 16, 16, 2, 128, 16, 1600, 16 * 912
    state, cache = list(ops.paged_kv_tables(R, 100, pages, dev)), ops.paged_kv_cache(pages, Hkv, ps, D, dev)
    want_lengths = torch.zeros(R, dtype=torch.int32, device=dev)
    qkv = torch.randn(1, T, (Hq + 2 * Hkv) * D, generator=g, device=dev).to(torch.bfloat16)
    q, k, v = (x.view(1, T, -1, D).transpose(1, 2) for x in qkv.split([Hq * D, Hkv * D, Hkv * D], -1))

    def step(state, cache):
        lengths, table, free, count = state
        new, left, starts, slots, _ = ops.paged_kv_resize(lengths, want_lengths, table, free, count, ps, T)
        ops.paged_kv_write(k, v, *cache, slots)
        out = ops.paged_attention(q, *cache, table, new, starts, causal=True)
        lengths.copy_(new)
        count.copy_(left)
        return out, starts

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([t.clone() for t in state], [t.clone() for t in cache])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, starts = step(state, cache)
    held = [0] * R
    for i, grow in enumerate((lambda r: 912, lambda r: 1, lambda r: 1, lambda r: rng.randint(0, 5), lambda r: 32, lambda r: 0, lambda r: 1 if r else 300, lambda r: 1)):
        held = [n + grow(r) for r, n in enumerate(held)]
        qkv.copy_(torch.randn(qkv.shape, generator=g, device=dev))
        want_lengths.copy_(ints(held, dev))
        graph.replay()
        assert state[0].tolist() == held
        check(out, wanted(q, cache, state[1], held, starts.tolist(), True), f"replay {i}")


def test_cuts_of_wide_tables(dev):
    """Tables that could hold 2^30 keys a request, of which some ten thousand are there: measures in hundreds of keys, cuts on items' ends."""
    rng, g = random.Random(6), torch.Generator(device=dev).manual_seed(6)
    ps, width, counts, lengths = 65536, 16383, [702, 263, 8, 5, 187, 7], [10691, 11389, 10062, 10170, 11209, 10193]
    cache = pool(6, 4, ps, 64, torch.bfloat16, True, g, dev)
    table = tables(lengths, ps, 6, 1, rng, dev)
    starts = prefix(counts)
    q = torch.randn(1, starts[-1] + 5, 16, 64, generator=g, device=dev).to(torch.bfloat16).transpose(1, 2)
    wide = torch.cat((table, table.new_full((6, width - 1), -1)), 1)
    out = ops.paged_attention(q, *cache, wide, ints(lengths, dev), ints(starts, dev), causal=True)
    check(out, wanted(q, cache, table, lengths, starts, True), "wide")


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,length", [(9, 5), (64, 40), (100, 60), (300, 170)])
def test_queries_before_the_first_key(dev, n, length, dtype, e4m3):
    """More queries than keys: those in front of the first key see nothing and get zeros, whatever the others see."""
    rng, g = random.Random(n), torch.Generator(device=dev).manual_seed(n)
    Hq, Hkv, D, ps = 2, 1, 64, 16
    cache = pool(30, Hkv, ps, D, dtype, e4m3, g, dev)
    table = tables([length], ps, 30, 20, rng, dev)
    q = torch.randn(1, n, Hq, D, generator=g, device=dev).to(dtype).transpose(1, 2)
    value, tol = wanted(q, cache, table, [length], [0, n], True)
    first = n - length  # the first query that sees a key
    page = int(table[0, 0])
    for odd in (float("nan"), float("inf")):
        bad = [None if t is None else t.clone() for t in cache]
        if not e4m3:
            bad[1][page, 0, 0, 5] = odd  # (of e4m3's codes only NaN is not finite)
        elif odd == float("inf"):
            bad[3][page, 0, 0] = odd     # a scale
        else:
            bad[1].view(torch.uint8)[page, 0, 0, 5] = 0x7F
        out = ops.paged_attention(q, *bad, table, ints([length], dev), ints([0, n], dev), causal=True)
        assert not out[0, :, :first].any(), "a query that sees nothing"  # (NaN counts as true)
        sees = torch.zeros_like(out, dtype=torch.bool)
        sees[0, :, first:] = True
        hit = sees.clone() if e4m3 and odd == float("inf") else sees & (torch.arange(D, device=dev) == 5)
        assert not bool(torch.isfinite(out[hit]).any())
        check(out.masked_fill(hit, 0), (value.masked_fill(hit, 0), tol), "what is finite")


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,length", [(1, 1), (1, 20), (5, 900), (1, 9000), (70, 200), (300, 3000)])
def test_a_request_whose_pages_are_all_none(dev, n, length, dtype, e4m3):
    """Zeros, though the pool's first slot, which another request owns, holds NaN and infinities."""
    Hq, Hkv, D, ps = 8, 2, 128, 16
    g = torch.Generator(device=dev).manual_seed(n)
    cache = pool(3, Hkv, ps, D, dtype, e4m3, g, dev)
    table = torch.full((2, -(-length // ps)), -1, dtype=torch.int32, device=dev)
    table[1, 0] = 0
    q = torch.randn(1, n + 1, Hq, D, generator=g, device=dev).to(dtype).transpose(1, 2)
    for odd in (float("nan"), float("inf")):
        for i in range(2):
            if e4m3:
                cache[i].view(torch.uint8)[0, :, 0] = 0x7F
                cache[2 + i][0, :, 0] = odd
            else:
                cache[i][0, :, 0] = odd
        for causal in (True, False):
            out = ops.paged_attention(q, *cache, table, ints([length, 1], dev), ints([0, n, n + 1], dev), causal=causal)
            assert not out[0, :, :n].any() and bool(torch.isnan(out[0, :, n]).all())


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,length", [(1, 100), (1, 300), (1, 30000), (40, 9000), (200, 12000)])
def test_a_value_that_is_none_counts_at_any_distance(dev, n, length, dtype, e4m3):
    """0 * NaN and 0 * infinity are no numbers: a value whose probability is 0 in 32 bits beside another's counts wherever its request is cut."""
    Hq, Hkv, D, ps = 8, 2, 128, 64
    pages = -(-length // ps)
    cache = list(ops.paged_kv_cache(pages, Hkv, ps, D, dev, *([] if e4m3 else [dtype])))
    for t in cache[2:] if e4m3 else ():
        t.fill_(1.0)
    cache[1].copy_(torch.randn(cache[1].shape, generator=torch.Generator(device=dev).manual_seed(1), device=dev))
    table = torch.arange(pages, dtype=torch.int32, device=dev)[None]
    q = torch.full((1, n, Hq, D), 8.0, dtype=dtype, device=dev).transpose(1, 2)
    cache[0][(length - n) // ps, :, (length - n) % ps] = 8.0  # scores 8 * 8 * sqrt(128) = 724 there, 0 elsewhere; all queries see it
    for odd in ([float("nan")] if e4m3 else [float("nan"), float("inf")]):
        cache[1][0, 1, 3, 7] = odd
        out = ops.paged_attention(q, *cache, table, ints([length], dev), ints([0, n], dev), causal=True)
        hit = torch.zeros_like(out, dtype=torch.bool)
        hit[0, Hq // 2:, :, 7] = True
        assert not bool(torch.isfinite(out[hit]).any()) and bool(torch.isfinite(out[~hit]).all())


def both_hosts(monkeypatch):
    yield "native host"
    monkeypatch.setattr(_lib, "_host", _lib._NoHost)
    yield "Python host"


def test_derivatives_of_the_pages_are_refused(dev, monkeypatch):
    """Pages and scales that need gradients or carry tangents, as queries, keys and values that do."""
    x = torch.randn(1, 2, 3, 64, device=dev).to(torch.bfloat16)
    table, lengths, starts, slots = ints([[0, 1]], dev), ints([20], dev), ints([0, 3], dev), ints([0, 1, 2], dev)
    for host in both_hosts(monkeypatch):
        for dtype in (torch.float8_e4m3fn, torch.bfloat16):
            cache = ops.paged_kv_cache(2, 2, 16, 64, dev, dtype)
            attend = lambda c: ops.paged_attention(x, *c, table, lengths, starts, causal=True)  # noqa: E731
            write = lambda c: ops.paged_kv_write(x, x, *c, slots)  # noqa: E731
            write(cache)
            want = attend(cache)
            for i, t in enumerate(cache):
                if t is None:
                    continue
                needs = [*cache[:i], t.clone().requires_grad_(), *cache[i + 1:]]
                for call in (attend, write):
                    with pytest.raises(RuntimeError, match="differentiable"):
                        call(needs)
                    with torch.no_grad():
                        call(needs)
                assert torch.equal(attend([None if y is None else y.detach() for y in needs]), want), host
                if dtype == torch.float8_e4m3fn and i < 2:
                    continue  # (codes carry no tangents)
                with torch.autograd.forward_ad.dual_level():
                    dual = [*cache[:i], torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)), *cache[i + 1:]]
                    for call in (attend, write):
                        with pytest.raises(RuntimeError, match="forward-mode"):
                            call(dual)


@pytest.mark.parametrize("max_tokens", [0, 5, 4096])
def test_resize_results_own_their_memory(dev, monkeypatch, max_tokens):
    """Each result alone in its memory, in both hosts: growing one leaves the others, saving one saves it alone."""
    for host in both_hosts(monkeypatch):
        lengths, table, free, count = ops.paged_kv_tables(3, 4, 12, dev)
        got = ops.paged_kv_resize(lengths, ints([1, 0, 4], dev), table, free, count, 16, max_tokens)
        for x in got:
            assert x.untyped_storage().nbytes() == x.numel() * x.element_size() and x.storage_offset() == 0 and x._base is None, host
        assert len({x.untyped_storage().data_ptr() for x in got if x.numel()}) == sum(x.numel() > 0 for x in got)
        before = [x.clone() for x in got]
        for i, x in enumerate(got):
            x.resize_(x.numel() + 100)[before[i].numel():].fill_(-9)
            assert all(torch.equal(y[: z.numel()], z) for y, z in zip(got, before)), host
        side = torch.cuda.Stream()
        for x in got:
            x.record_stream(side)


def test_more_tokens_than_max_tokens(dev):
    """They show in starts, and the call made again with room for them is as if it had been the first."""
    for wanted_ in ([9, 3, 40, 0], [9, 3, 1000, 30]):  # (of 12 pages; of more than there are)
        state, other = ops.paged_kv_tables(4, 20, 12, dev), ops.paged_kv_tables(4, 20, 12, dev)
        short = ops.paged_kv_resize(state[0], ints(wanted_, dev), *state[1:], 4, 11)
        grown = int((short[0] - state[0]).clamp(min=0).sum())
        assert int(short[2][-1]) == 11 < grown and int((short[3] >= 0).sum()) == 11
        again, first = (ops.paged_kv_resize(s[0], ints(wanted_, dev), *s[1:], 4, 60) for s in (state, other))
        assert all(torch.equal(a, b) for a, b in zip(again, first)) and int(again[2][-1]) == grown
        for r, n in enumerate(again[0].tolist()):  # (what a request owns)
            assert torch.equal(state[1][r, : -(-n // 4)], other[1][r, : -(-n // 4)])


def test_nothing_to_attend_to_in_pages_that_hold_something(dev):
    g = torch.Generator(device=dev).manual_seed(2)
    q = torch.randn(1, 9, 4, 64, generator=g, device=dev).to(torch.bfloat16).transpose(1, 2)
    none, zero = torch.zeros(0, 5, dtype=torch.int32, device=dev), ints([[0]] * 3, dev)
    for e4m3 in (True, False):
        cache = pool(3, 2, 16, 64, torch.bfloat16, e4m3, g, dev)
        for causal in (True, False):
            attend = lambda *args: ops.paged_attention(q, *cache, *args, causal=causal)  # noqa: E731
            assert attend(ints([[0]], dev), ints([9], dev)).any()
            assert not attend(none, ints([], dev), ints([4], dev)).any()                                                      # no requests
            assert not attend(zero, ints([0, -5, 0], dev), ints([0, 4, 4, 9], dev)).any()                                     # no keys
            assert not attend(zero, ints([9, 9, 9], dev), ints([4, 4, 4, 4], dev)).any()                                      # no queries
            assert not attend(torch.zeros(3, 0, dtype=torch.int32, device=dev), ints([9, 9, 9], dev), ints([0, 4, 4, 9], dev)).any()  # no pages to a request


@pytest.mark.parametrize("e4m3", [True, False])
def test_requests_that_claim_the_same_tokens(dev, e4m3):
    """Whatever stands in their tokens, nothing else is written; of more work than any requests that ascend can ask for nothing is done."""
    rng, g = random.Random(3), torch.Generator(device=dev).manual_seed(3)
    cache = pool(40, 1, 16, 64, torch.bfloat16, e4m3, g, dev)
    for R, T, Hq, most in ((7, 300, 2, 500), (200, 4096, 8, 2000), (60, 9000, 4, 90), (600, 700, 1, 600)):
        table = torch.randint(0, 40, (R, most // 16 + 1), generator=g, device=dev).to(torch.int32)
        lengths, starts = ([rng.randint(0, most) for _ in range(R)], [rng.randint(-3, T + 3) for _ in range(R + 1)])
        q = torch.randn(1, T, Hq, 64, generator=g, device=dev).to(torch.bfloat16).transpose(1, 2)
        for causal in (True, False):
            guarded(q, cache, table, ints(lengths, dev), ints(starts, dev), causal)
    R, T, width = 4600, 4096, 512
    q = torch.randn(1, T, 1, 64, generator=g, device=dev).to(torch.bfloat16).transpose(1, 2)
    args = (torch.zeros(R, width, dtype=torch.int32, device=dev), ints([width * 16] * R, dev))
    assert guarded(q, cache, *args, ints([min(r, T) for r in range(R + 1)], dev), False).any()
    assert not guarded(q, cache, *args, ints([T * (r % 2) for r in range(R + 1)], dev), False).any()


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("n", [2, 70])
def test_pools_of_more_than_2_32_values(dev, n, e4m3):
    """Pages on either side of 2^31 and 2^32 values into the pool, written through slots and read."""
    Hq, Hkv, D, ps, dtype = 8, 4, 128, 256, torch.bfloat16
    pages, g = 2 ** 32 // (Hkv * D * ps) + 9, torch.Generator(device=dev).manual_seed(n)
    cache = [torch.empty(pages, Hkv, ps, D, dtype=torch.float8_e4m3fn if e4m3 else dtype, device=dev) for _ in range(2)]
    cache += [torch.empty(pages, Hkv, ps, dtype=torch.float32, device=dev) if e4m3 else None for _ in range(2)]
    half = pages // 2
    table, lengths = ints([[pages - 1, half, 3], [half - 6, pages - 9, pages - 3]], dev), [700, 513]
    at = torch.arange(max(lengths), device=dev)
    slots = torch.cat([table[r].long()[at[:x] // ps] * ps + at[:x] % ps for r, x in enumerate(lengths)]).to(torch.int32)
    k, v = (torch.randn(1, slots.numel(), Hkv, D, generator=g, device=dev).to(dtype).transpose(1, 2) for _ in range(2))
    ops.paged_kv_write(k, v, *cache, slots)
    own = [None if t is None else t[table.flatten().long()] for t in cache]
    small = torch.arange(6, dtype=torch.int32, device=dev).view(2, 3)
    q = torch.randn(1, 2 * n, Hq, D, generator=g, device=dev).to(dtype).transpose(1, 2)
    out = ops.paged_attention(q, *cache, table, ints(lengths, dev), ints([0, n, 2 * n], dev), causal=True)
    check(out, wanted(q, own, small, lengths, [0, n, 2 * n], True), "large pool")
    flat = torch.cat([own[1][r * 3 + at[:x] // ps, :, at[:x] % ps].double() * (own[3][r * 3 + at[:x] // ps, :, at[:x] % ps].double()[..., None] if e4m3 else 1) for r, x in enumerate(lengths)])
    # (e4m3: a code is off by half a step, 2^-4 of the value or, below the least normal code, 2^-10 of the scale, a 448th of a row's largest value, which is below 8)
    assert bool(((flat - v[0].transpose(0, 1).double()).abs() <= (v[0].transpose(0, 1).double().abs() * 2 ** -4 + 2 ** -10 * 8 / 448 if e4m3 else 0)).all())


@pytest.mark.parametrize("Hq,Hkv", [(1024, 1), (100, 1), (66, 2)])
def test_many_query_heads_to_a_key_head(dev, Hq, Hkv):
    """Groups of more heads than a tile has rows."""
    rng, g = random.Random(Hq), torch.Generator(device=dev).manual_seed(Hq)
    counts, lengths = [1, 2, 0, 3], [70, 1300, 9, 200]
    cache = pool(120, Hkv, 16, 64, torch.bfloat16, True, g, dev)
    table, starts = tables(lengths, 16, 120, 90, rng, dev), prefix(counts)
    q = torch.randn(1, 7, Hq, 64, generator=g, device=dev).to(torch.bfloat16).transpose(1, 2)
    for causal in (True, False):
        out = ops.paged_attention(q, *cache, table, ints(lengths, dev), ints(starts, dev), causal=causal)
        check(out, wanted(q, cache, table, lengths, starts, causal), "group")


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("n", [3, 100])
def test_queries_that_are_no_numbers(dev, n, e4m3):
    """A query of NaN is its own affair; queries that lie in memory as one do, seen through strides of 0, are many."""
    rng, g = random.Random(n), torch.Generator(device=dev).manual_seed(n)
    lengths, starts = [n + 500, n + 30], [0, n, 2 * n]
    cache = pool(120, 2, 16, 128, torch.bfloat16, e4m3, g, dev)
    table = tables(lengths, 16, 120, 60, rng, dev)
    q = torch.randn(1, 2 * n, 8, 128, generator=g, device=dev).to(torch.bfloat16).transpose(1, 2)
    args = (*cache, table, ints(lengths, dev), ints(starts, dev))
    clean = ops.paged_attention(q, *args, causal=True)
    odd = q.clone()
    odd[0, 2, 1, 7], odd[0, 5, n, 0] = float("nan"), float("nan")
    out = ops.paged_attention(odd, *args, causal=True)
    assert bool(torch.isnan(out[0, 2, 1]).all()) and bool(torch.isnan(out[0, 5, n]).all())
    out[0, 2, 1], out[0, 5, n] = clean[0, 2, 1], clean[0, 5, n]
    assert torch.equal(out, clean)
    same = q[:, :1, :1].expand(1, 8, 2 * n, 128)
    assert torch.equal(ops.paged_attention(same, *args, causal=True), ops.paged_attention(same.contiguous(), *args, causal=True))
