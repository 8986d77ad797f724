"""A paged key / value cache, as cases that can be timed and compared: the block tables and slot maps of requests that
grow, shrink and end, the write of new tokens through a slot map, and attention of the requests' new tokens (one token,
a few drafted ones, a denoise step's action tokens, chunks of a prompt) over the pages.

The cache is a pool of pages [pages, Hkv, page size, D], e4m3 with a scale per token and head or in the tokens' own type.
Request r holds lengths[r] tokens; token i of it lies in page page_table[r, i // page size] at i % page size.  Tokens of
all requests stand behind each other: request r's new ones are starts[r] .. starts[r + 1] - 1.

Sizes are those of the repository's own configurations (`wallx_mi355.workloads`: 16 query and 2 key / value heads of 128,
rows of 912 tokens with 32 action tokens; heads of 64 and 80 elsewhere) and generic ones.  With `own` false `run` computes
a case in its plain form, in fp32 with one rounding at the end; with `own` true through the framework's ops.

  tables   pages given to growing requests and taken back from shrinking ones, slots and positions of the new tokens
  write    new keys and values into their slots, quantised or as they are
  attn     attention of the new tokens over their requests' pages
"""

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
F8 = torch.float8_e4m3fn
F8_MAX, SCALE_MIN = 448.0, 2.0 ** -126


def _ops():
    path = os.path.abspath("wall-x_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from wallx_mi355.fusions import ops

    return ops


def listed():
    heads = dict(Hq=16, Hkv=2, D=128, dtype="bf16")
    return [
        # a generation step of 64 requests, a token each: the call's latency
        dict(name="tables_step_64", kind="tables", R=64, P=128, ps=16, held_lo=1, held_hi=2000, grow=1, ends=0.0, joins=0.0),
        # a busy server between two steps: 1000 requests, some end, others join with their prompts, the rest take a token
        dict(name="tables_turnover_1000", kind="tables", R=1000, P=256, ps=16, held_lo=0, held_hi=4000, grow=1, ends=0.1, joins=0.1),
        # that step's tokens into the e4m3 cache
        dict(name="write_step_64", kind="write", R=64, S=1, ps=16, Hkv=2, D=128, dtype="bf16", cache="e4m3", pad=0),
        # prompts of 16 rows of 912 tokens
        dict(name="write_prompts_16", kind="write", R=16, S=912, ps=64, Hkv=2, D=128, dtype="bf16", cache="e4m3", pad=0),
        # an odd number of tokens of eight heads of 80 into a cache of their own type, padding behind the last request
        dict(name="write_plain_5003", kind="write", R=3, S=5003, ps=48, Hkv=8, D=80, dtype="fp16", cache="same", pad=77),
        # single-token generation of 64 robots over their prefixes
        dict(name="attn_step_64", kind="attn", R=64, n=1, ragged=False, big=0, chunk=0, past_lo=800, past_hi=912, ps=16, cache="e4m3", causal=True, pad=0, **heads),
        # single-token generation over long ragged contexts
        dict(name="attn_step_32k", kind="attn", R=8, n=1, ragged=False, big=0, chunk=0, past_lo=20001, past_hi=32768, ps=16, cache="e4m3", causal=True, pad=0, **heads),
        # up to five drafted tokens of 32 requests checked at once, cache in bf16
        dict(name="attn_drafts_32", kind="attn", R=32, n=5, ragged=True, big=0, chunk=0, past_lo=0, past_hi=16000, ps=64, cache="same", causal=True, pad=8, **heads),
        # a denoise step of 64 robots: 32 action queries that see the prefix and each other
        dict(name="attn_denoise_64", kind="attn", R=64, n=32, ragged=False, big=0, chunk=0, past_lo=768, past_hi=880, ps=16, cache="e4m3", causal=False, pad=0, **heads),
        # a chunk of a long prompt over what is in the cache of it
        dict(name="attn_chunk_2048", kind="attn", R=1, n=1, ragged=False, big=1, chunk=2048, past_lo=14336, past_hi=14336, ps=64, cache="e4m3", causal=True, pad=0, **heads),
        # a mixed batch: two chunks of prompts among 62 requests that take a token; 14 / 2 heads of 64 in fp16
        dict(name="attn_mixed_64", kind="attn", R=64, n=1, ragged=False, big=2, chunk=509, past_lo=100, past_hi=4000, ps=32, cache="e4m3", causal=True, pad=3,
             Hq=14, Hkv=2, D=64, dtype="fp16"),
        # whole prompts of 16 rows at once, nothing before them, cache in bf16
        dict(name="attn_prompts_16", kind="attn", R=16, n=1, ragged=False, big=16, chunk=912, past_lo=0, past_hi=0, ps=128, cache="same", causal=True, pad=0, **heads),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["tables", "write", "attn", "attn", "attn"])
    ps = rng.choice([8, 16, 16, 32, 48, 64, 128, 256])
    if kind == "tables":
        R = _log(rng, 1, 2000)
        P = _log(rng, 2, max(2, min(1024, 4000000 // (R * ps))))
        return dict(kind=kind, R=R, P=P, ps=ps, held_lo=0, held_hi=max(1, rng.randrange(1, P * ps + 1)), grow=_log(rng, 1, 64),
                    ends=rng.choice([0.0, 0.1, 0.5]), joins=rng.choice([0.0, 0.1]))
    Hkv = rng.choice([1, 2, 4, 8])
    D = rng.choice([64, 80, 128])
    dtype, cache = rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["e4m3", "e4m3", "same"])
    if kind == "write":
        tokens = _log(rng, 1, 60000 // Hkv)
        R = min(tokens, _log(rng, 1, 128))
        return dict(kind=kind, R=R, S=tokens // R, ps=ps, Hkv=Hkv, D=D, dtype=dtype, cache=cache, pad=rng.choice([0, 0, rng.randrange(1, 65)]))
    Hq = Hkv * rng.choice([1, 2, 3, 4, 7, 8])
    form = rng.choice(["steps", "drafts", "chunks", "mixed"])
    past = _log(rng, 16, 32768)
    chunk = _log(rng, 9, 1024) if form in ("chunks", "mixed") else 0
    most = min(1.2e8 / (Hkv * (past + chunk) * D), 1.6e8 / (Hq * max(chunk, 8) * (past + chunk)))
    R = _log(rng, 1, int(max(1, min(192, most))))
    return dict(kind=kind, R=R, n=1 if form == "steps" else rng.randrange(2, 9), ragged=rng.random() < 0.5, big=R if form == "chunks" else min(R, 2) if form == "mixed" else 0,
                chunk=chunk, past_lo=rng.choice([0, past // 2]), past_hi=past, ps=ps, cache=cache, causal=rng.random() < 0.75, pad=rng.choice([0, 5]),
                Hq=Hq, Hkv=Hkv, D=D, dtype=dtype)


# ----------------------------------------------------------------------------- inputs
def _pages(tokens, ps):
    return -(-tokens // ps)


def _quantise(x):
    scale = (x.float().abs().amax(-1) / F8_MAX).clamp(min=SCALE_MIN)
    return (x.float() / scale[..., None]).to(F8), scale


def _pool(c, pages, g):
    """The pages' contents [pages, Hkv, page size, D] of keys and of values, with their scales or None."""
    out = {}
    for n in ("k", "v"):
        x = torch.randn(pages, c["Hkv"], c["ps"], c["D"], device="cuda", generator=g) * 2
        out[n + "_pages"], out[n + "_scale"] = _quantise(x) if c["cache"] == "e4m3" else (x.to(DTYPES[c["dtype"]]), None)
    return out


def _prompt_tokens(c):
    """A step's room for tokens of joining requests."""
    return int(c["R"] * c["joins"] * c["P"] * c["ps"] / 2)


def _table(counts, width, order):
    """page_table int32 [R, width]: request r's counts[r] pages, off the list `order`; -1 behind them."""
    rows, at = [], 0
    for n in counts:
        rows.append(order[at: at + n] + [-1] * (width - n))
        at += n
    return torch.tensor(rows, dtype=torch.int32, device="cuda").view(len(counts), width)


def prepare(case, seed):
    c, rng = case, random.Random(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    if c["kind"] == "tables":
        R, most = c["R"], c["P"] * c["ps"]
        held = [rng.randint(min(c["held_lo"], c["held_hi"]), min(c["held_hi"], most)) for _ in range(R)]
        want, room = [], _prompt_tokens(c)
        for h in held:
            x = rng.random()
            if x < c["ends"]:
                want.append(0)
            elif x < c["ends"] + c["joins"]:  # (as far as a step's room for prompts goes)
                want.append(h + min(room, rng.randint(0, most - h)))
                room -= want[-1] - h
            else:
                want.append(min(most, h + (c["grow"] if c["grow"] < 2 else rng.randint(1, c["grow"]))))
        counts = [_pages(h, c["ps"]) for h in held]
        pages = R * (_pages(min(c["held_hi"], most), c["ps"]) + 1)  # (joining requests may not find enough of them)
        order = list(range(pages))
        rng.shuffle(order)
        used = sum(counts)
        s["lengths"], s["wanted"] = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (held, want))
        s["page_table"] = _table(counts, c["P"], order)
        s["free_pages"] = torch.tensor(order[used:] + [-1] * used, dtype=torch.int32, device="cuda")
        s["free_count"] = torch.tensor([pages - used], dtype=torch.int32, device="cuda")
        s["tokens"] = R * c["grow"] + _prompt_tokens(c)
        return s
    dt, R, ps, Hkv, D = DTYPES[c["dtype"]], c["R"], c["ps"], c["Hkv"], c["D"]
    if c["kind"] == "write":
        each = _pages(c["S"], ps)
        pages = R * each + 8
        order = list(range(pages))
        rng.shuffle(order)
        table = _table([each] * R, each, order)
        at = torch.arange(c["S"], device="cuda")
        slots = (table[:, at // ps] * ps + at % ps).view(-1)
        s["slots"] = torch.cat((slots, slots.new_full((c["pad"],), -1))).to(torch.int32)
        s.update(_pool(c, pages, g))
        T = R * c["S"] + c["pad"]
        kv = torch.randn(1, T, 2 * Hkv * D, device="cuda", generator=g).to(dt)  # the projection's result
        s["k"], s["v"] = (x.view(1, T, Hkv, D).transpose(1, 2) for x in kv.split(Hkv * D, -1))
        return s
    chunks = [c["chunk"] if r < c["big"] else rng.randint(0, c["n"]) if c["ragged"] else c["n"] for r in range(R)]
    rng.shuffle(chunks)
    lengths = [n + rng.randint(c["past_lo"], c["past_hi"]) for n in chunks]
    counts = [_pages(x, ps) for x in lengths]
    pages = sum(counts) + 8
    order = list(range(pages))
    rng.shuffle(order)
    s["page_table"] = _table(counts, max(1, max(counts)), order)
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s["starts"] = torch.tensor([sum(chunks[:r]) for r in range(R + 1)], dtype=torch.int32, device="cuda")
    s["chunks"], s["held"] = chunks, lengths  # what the program scheduled
    s.update(_pool(c, pages, g))
    T = (R - c["big"]) * c["n"] + c["big"] * c["chunk"] + c["pad"]  # what a step has room for
    qkv = torch.randn(1, T, (c["Hq"] + 2 * Hkv) * D, device="cuda", generator=g).to(dt)
    s["q"] = qkv[..., : c["Hq"] * D].view(1, T, c["Hq"], D).transpose(1, 2)
    return s


# ----------------------------------------------------------------------------- the plain forms
def _plain_tables(s):
    """Freed pages go onto the list's end so that the first of them (by request, then by place) is the next one taken;
    growing requests take theirs off its end in the same order.  A request that the pages do not suffice for gets the
    tokens that it has pages for."""
    c = s["case"]
    ps, P, R = c["ps"], c["P"], c["R"]
    held, want, table = s["lengths"].long(), s["wanted"].long(), s["page_table"]
    free, count = s["free_pages"], s["free_count"].long()
    have, need = (held + ps - 1) // ps, (want + ps - 1) // ps
    give, take = (have - need).clamp(min=0), (need - have).clamp(min=0)
    given, taken = give.cumsum(0), take.cumsum(0)
    n_given = given[-1:]
    top = count + n_given
    got = (top - (taken - take)).clamp(min=0).minimum(take)
    new = torch.where(got < take, torch.minimum(want, (have + got) * ps), want)
    place = torch.arange(P, device="cuda")
    # of every page that is freed: its number in the order above, and the page
    freed = (place >= need[:, None]) & (place < have[:, None])
    number = torch.where(freed, (given - give)[:, None] + place - need[:, None], 0)
    by_number = torch.full((R * P + 1,), -1, dtype=torch.int32, device="cuda")
    by_number.scatter_(0, torch.where(freed, number, R * P).view(-1), table.reshape(-1))
    granted = (place >= have[:, None]) & (place < (have + got)[:, None])
    nth = (taken - take)[:, None] + place - have[:, None]
    fresh = torch.where(nth < n_given, by_number[nth.clamp(0, R * P)], free[(top - 1 - nth).clamp(0, free.numel() - 1)])
    table.copy_(torch.where(granted, fresh, table))
    n_taken = got.sum(0, keepdim=True)
    left = top - n_taken
    at = torch.arange(free.numel(), device="cuda")
    back = (at >= count) & (at < left)
    free.copy_(torch.where(back, by_number[(top - 1 - at).clamp(0, R * P)], free))
    added = (new - held).clamp(min=0)
    starts = torch.cat((added.new_zeros(1), added.cumsum(0)))
    token = torch.arange(s["tokens"], device="cuda")
    r = torch.searchsorted(starts, token, right=True).sub(1).clamp(max=R - 1)
    position = held[r] + token - starts[r]
    live = token < starts[-1]
    position = torch.where(live, position, 0)
    slots = torch.where(live, table[r, position // ps] * ps + position % ps, -1)
    return {"lengths": new.int(), "free_count": left.int(), "starts": starts.int(), "slots": slots.int(), "positions": position,
            "page_table": table, "free_pages": free}


def _plain_write(s):
    c = s["case"]
    page, at = torch.div(s["slots"], c["ps"], rounding_mode="floor").long(), (s["slots"] % c["ps"]).long()
    t = (s["slots"] >= 0).nonzero(as_tuple=True)[0]
    for n in ("k", "v"):
        x = s[n][0].transpose(0, 1)[t]
        if c["cache"] == "e4m3":
            x, scale = _quantise(x)
            s[n + "_scale"][page[t], :, at[t]] = scale
            s[n + "_pages"].view(torch.uint8)[page[t], :, at[t]] = x.view(torch.uint8)
        else:
            s[n + "_pages"][page[t], :, at[t]] = x


def _cache(s):
    return {n: s[n] for n in ("k_pages", "v_pages", "k_scale", "v_scale") if s[n] is not None}


def _gathered(s, n, rows, longest):
    """fp32 keys or values [requests, Hkv, tokens, D] of some requests, up to a number of tokens."""
    c = s["case"]
    table = s["page_table"][rows, : _pages(max(1, longest), c["ps"])].clamp(min=0).long()
    x = s[n + "_pages"][table].float()
    if s[n + "_scale"] is not None:
        x = x * s[n + "_scale"][table][..., None]
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attn(s):
    c = s["case"]
    group, T = c["Hq"] // c["Hkv"], s["q"].size(2)
    out = torch.zeros(T + 1, c["Hq"], c["D"], device="cuda", dtype=DTYPES[c["dtype"]])
    few = [r for r, n in enumerate(s["chunks"]) if 0 < n <= 8]
    sets = [few] if few else []  # requests of a like number of tokens together, as far as their scores' memory goes
    at_once = int(max(1, 3e8 // (max(max(s["chunks"]), 1) * max(s["held"] + [1]) * c["Hq"])))
    many = [r for r, n in enumerate(s["chunks"]) if n > 8]
    for requests in sets + [many[i: i + at_once] for i in range(0, len(many), at_once)]:
        if len(requests) == c["R"]:
            rows = slice(None)
        else:
            rows = torch.tensor(requests, device="cuda")
        longest, most = max(s["held"][r] for r in requests), max(s["chunks"][r] for r in requests)
        k, v = _gathered(s, "k", rows, longest), _gathered(s, "v", rows, longest)
        m, i = len(requests), torch.arange(most, device="cuda")
        first, count, end = s["starts"][:-1][rows].long()[:, None], s["starts"].diff()[rows][:, None], s["lengths"][rows][:, None]
        token = torch.where(i < count, first + i, T)
        q = s["q"][0].transpose(0, 1)[token.clamp(max=max(T - 1, 0))].float()  # [requests, queries, Hq, D]
        q = q.view(m, most, c["Hkv"], group, c["D"]).permute(0, 2, 3, 1, 4).reshape(m, c["Hkv"], group * most, c["D"])
        p = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(c["D"])).view(m, c["Hkv"], group, most, -1)
        last = end - count + i + 1 if c["causal"] else end.expand(m, most)
        p.masked_fill_((torch.arange(k.size(2), device="cuda") >= torch.minimum(last, end)[..., None])[:, None, None], -math.inf)
        p.sub_(p.amax(-1, keepdim=True).clamp_(min=-3e38)).exp_()
        p.div_(p.sum(-1, keepdim=True).clamp_(min=1e-38))
        y = torch.matmul(p.view(m, c["Hkv"], group * most, -1), v).view(m, c["Hkv"], group, most, c["D"])
        out[token] = y.permute(0, 3, 1, 2, 4).reshape(m, most, c["Hq"], c["D"]).to(out.dtype)
    return {"out": out[:T].transpose(0, 1)[None]}


def run(state):
    s, c = state, state["case"]
    if own:
        return _own(s, c)
    if c["kind"] == "tables":
        return _plain_tables(s)
    if c["kind"] == "write":
        _plain_write(s)
        return _cache(s)
    return _plain_attn(s)


def _own(s, c):
    ops = _ops()
    if c["kind"] == "tables":
        made = ops.paged_kv_resize(s["lengths"], s["wanted"], s["page_table"], s["free_pages"], s["free_count"], c["ps"], s["tokens"])
        return {**dict(zip(("lengths", "free_count", "starts", "slots", "positions"), made)), "page_table": s["page_table"], "free_pages": s["free_pages"]}
    if c["kind"] == "write":
        ops.paged_kv_write(s["k"], s["v"], s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"], s["slots"])
        return _cache(s)
    return {"out": ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"], s["page_table"], s["lengths"], s["starts"], causal=c["causal"])}


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    if c["kind"] == "tables":
        most = c["P"] * c["ps"]
        held = (c["held_lo"] + min(c["held_hi"], most)) / 2
        tokens = c["R"] * (c["joins"] * (most - held) / 2 + (1 - c["joins"] - c["ends"]) * (c["grow"] + 1) / 2)
        pages = tokens / c["ps"] + c["R"] * c["ends"] * held / c["ps"]
        # lengths and sizes in and out, pages from one list to the other, a slot and a position a token
        return {"bytes": 16 * c["R"] + 8 * pages + 12 * tokens, "flops": 4 * tokens}
    e = 1 if c["cache"] == "e4m3" else 2
    stored = c["D"] * e + (4 if e == 1 else 0)
    if c["kind"] == "write":
        rows = 2 * c["R"] * c["S"] * c["Hkv"]
        return {"bytes": rows * (2 * c["D"] + stored) + 4 * c["R"] * c["S"], "flops": 4 * rows * c["D"]}
    small, n = c["R"] - c["big"], (c["n"] / 2 if c["ragged"] else c["n"])
    past, tokens = (c["past_lo"] + c["past_hi"]) / 2, small * n + c["big"] * c["chunk"]
    keys = c["R"] * past + tokens
    pairs = sum(r * x * (past + ((x + 1) / 2 if c["causal"] else x)) for r, x in ((small, n), (c["big"], c["chunk"])))
    return {"bytes": 4 * tokens * c["Hq"] * c["D"] + 2 * keys * c["Hkv"] * stored, "flops": 4 * pairs * c["Hq"] * c["D"]}


# ----------------------------------------------------------------------------- in 64 bits, from the definition
def exact(case, seed):
    c = case
    if c["kind"] != "attn":
        return None  # whole numbers, codes and copies are what they are
    if c["R"] * c["Hq"] > 4096:
        return None
    s = prepare(case, seed)
    group, T, ps = c["Hq"] // c["Hkv"], s["q"].size(2), c["ps"]
    out = torch.zeros(1, c["Hq"], T, c["D"], device="cuda", dtype=torch.float64)
    first = 0
    for r, (n, length) in enumerate(zip(s["chunks"], s["held"])):
        if n == 0 or length == 0:
            continue
        token = torch.arange(length, device="cuda")
        page = s["page_table"][r].long()[token // ps]
        position = length - n + torch.arange(n, device="cuda")  # of the queries
        for hk in range(c["Hkv"]):
            k, v = (s[x + "_pages"][page, hk, token % ps].double() for x in "kv")
            if c["cache"] == "e4m3":
                k, v = (x * s[name][page, hk, token % ps].double()[:, None] for x, name in ((k, "k_scale"), (v, "v_scale")))
            for h in range(hk * group, (hk + 1) * group):
                score = s["q"][0, h, first: first + n].double() @ k.t() / math.sqrt(c["D"])
                if c["causal"]:
                    score = score.masked_fill(token > position[:, None], -math.inf)
                out[0, h, first: first + n] = torch.exp(score - torch.logsumexp(score, 1, keepdim=True)) @ v
        first += n
    return {"out": out}
