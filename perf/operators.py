"""A decoder layer's attention, as cases that can be timed and compared: the norm of q and k per head with the rotary
embedding, attention under a mask of key ranges with its gradients, and the quantised key / value cache with the
attention that reads it.

Sizes are those of the repository's own configurations (`wallx_mi355.workloads`: 16 query and 2 key / value heads of
128, rows of 912 tokens with 32 action tokens at their end, mrope_section [16, 24, 24]; the vision tower's 16 heads of
80 over windows of 64 patches) and generic ones.  With `own` false `run` computes a case in its plain form, in fp32 with
one rounding at the end; with `own` true through the framework's ops.

  qknorm   RMS norm per head and rotary embedding of q and k; with grad the gradients of q, k and both weights
  attn     attention; with grad the gradients of q, k and v
  write    a cache's keys and values quantised as they are written
  cached   attention of a few queries over the quantised cache
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
F8 = torch.float8_e4m3fn
F8_MAX, SCALE_MIN = 448.0, 2.0 ** -126
THETA, EPS = 1.0e6, 1e-6


def _ops():
    path = os.path.abspath("wall-x_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from wallx_mi355.fusions import ops

    return ops


def listed():
    return [
        # one generated token of each of 64 sequences: next to no work, the call's latency
        dict(name="qk_step_64", kind="qknorm", B=64, S=1, Hq=16, Hkv=2, D=128, dtype="bf16", src="table", layout="hf", far=4096, grad=False),
        # a training batch of 16 rows, forward and backward
        dict(name="qk_train_16", kind="qknorm", B=16, S=912, Hq=16, Hkv=2, D=128, dtype="bf16", src="table", layout="hf", far=0, grad=True),
        # fp32 heads of 64 at far positions, an odd number of tokens, the angles evaluated from the position ids
        dict(name="qk_train_fp32", kind="qknorm", B=3, S=1237, Hq=14, Hkv=2, D=64, dtype="fp32", src="positions", layout="csrc", far=30000, grad=True),
        # a prefill of 16 rows: causal with the action block, some rows padded on the left
        dict(name="attn_prefill_16", kind="attn", B=16, Sq=912, Sk=912, Hq=16, Hkv=2, D=128, dtype="bf16", mask="action", grad=False),
        # one long causal sequence
        dict(name="attn_causal_16k", kind="attn", B=1, Sq=16384, Sk=16384, Hq=16, Hkv=2, D=128, dtype="bf16", mask="causal", grad=False),
        # the vision tower's windows: 48 camera images of 32 x 32 patches, 64 patches a window, heads of 80
        dict(name="attn_windows_48", kind="attn", B=48, Sq=1024, Sk=1024, Hq=16, Hkv=16, D=80, dtype="fp16", mask="windows", grad=False),
        # a training batch of 16 rows with the action block, forward and backward
        dict(name="attn_train_16", kind="attn", B=16, Sq=912, Sk=912, Hq=16, Hkv=2, D=128, dtype="bf16", mask="action", grad=True),
        # sequences packed into one row of odd length, forward and backward
        dict(name="attn_train_packed", kind="attn", B=1, Sq=5003, Sk=5003, Hq=12, Hkv=4, D=64, dtype="fp16", mask="packed", grad=True),
        # the prefix of 64 robots into the cache after a prefill
        dict(name="write_prefix_64", kind="write", B=64, S=880, C=1024, Hkv=2, D=128, dtype="bf16", ragged=True),
        # one generated token of each of 64 sequences into a long cache
        dict(name="write_step_64", kind="write", B=64, S=1, C=8192, Hkv=2, D=128, dtype="bf16", ragged=False),
        # a denoise step of 64 robots: 32 action queries over the prefix and themselves
        dict(name="cached_denoise_64", kind="cached", B=64, Sq=32, C=1024, Hq=16, Hkv=2, D=128, dtype="bf16", shortest=800, longest=912, causal=False),
        # single-token generation over long ragged caches
        dict(name="cached_decode_32k", kind="cached", B=8, Sq=1, C=32768, Hq=16, Hkv=2, D=128, dtype="bf16", shortest=20001, longest=32768, causal=True),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["qknorm", "attn", "attn", "write", "cached"])
    Hkv = rng.choice([1, 2, 4, 8])
    Hq = Hkv * rng.choice([1, 2, 3, 4, 7, 8])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "qknorm":
        src = rng.choice(["table", "positions"])
        tokens = _log(rng, 1, 30000)
        B = min(tokens, _log(rng, 1, 64))
        return dict(kind=kind, B=B, S=max(1, min(tokens // B, 300000 // (B * (Hq + Hkv)))), Hq=Hq, Hkv=Hkv, D=rng.choice([64, 128]),
                    dtype="bf16" if src == "table" else rng.choice(["bf16", "fp16", "fp32"]), src=src, layout=rng.choice(["hf", "csrc"]),
                    far=rng.choice([0, rng.randrange(1, 100000)]), grad=rng.random() < 0.6)
    if kind == "attn":
        mask = rng.choice(["action", "causal", "packed", "full", "windows"])
        grad = rng.random() < 0.6
        S = _log(rng, 1, 8192)
        Sk = S + rng.choice([0, _log(rng, 1, 2000)]) if mask in ("causal", "full") else S
        B = _log(rng, 1, max(1, min(64, int((4.0e8 if grad else 1.0e9) / (Hq * S * Sk)))))
        return dict(kind=kind, B=B, Sq=S, Sk=Sk, Hq=Hq, Hkv=Hkv, D=rng.choice([64, 80, 128]), dtype=dtype, mask=mask, grad=grad)
    D = rng.choice([64, 80, 128])
    C = _log(rng, 64, 65536)
    if kind == "write":
        S = _log(rng, 1, C)
        B = _log(rng, 1, max(1, min(128, int(1.0e5 / C))))
        return dict(kind=kind, B=B, S=S, C=C, Hkv=Hkv, D=D, dtype=dtype, ragged=rng.random() < 0.5)
    Sq = rng.choice([1, 1, _log(rng, 1, 64)])
    B = _log(rng, 1, max(1, min(128, int(min(3.0e5 / C, 1.2e8 / (Hkv * C * D), 6.0e8 / (Hq * Sq * C))))))
    return dict(kind=kind, B=B, Sq=Sq, C=C, Hq=Hq, Hkv=Hkv, D=D, dtype=dtype, shortest=rng.choice([0, C // 2]), longest=C, causal=rng.random() < 0.5)


# ----------------------------------------------------------------------------- inputs
def _section(D):
    return [D // 8, D // 16 * 3, D // 16 * 3]  # [16, 24, 24] for 128


def _planes(D, layout):
    """Which of the (t, h, w) position planes each channel takes."""
    s = _section(D)
    per = [0] * s[0] + [1] * s[1] + [2] * s[2]
    return per + per if layout == "hf" else [0] * (2 * s[0]) + [1] * (2 * s[1]) + [2] * (2 * s[2])


def _key_ranges(c, g):
    """lo, hi int32 [B, Sq]: the keys that a query may see, [lo, hi); None where the mask needs none."""
    B, S = c["B"], c["Sq"]
    i = torch.arange(S, device="cuda")
    if c["mask"] == "action":  # causal, the action tokens at the row's end see each other; every other row padded on the left
        pad = torch.randint(0, S // 4 + 1, (B, 1), device="cuda", generator=g) * (torch.arange(B, device="cuda")[:, None] % 2)
        act = min(32, S - S // 4)
        hi = torch.where(i >= S - act, S, i + 1).expand(B, S)
        lo = pad.expand(B, S)
        hi = torch.where(i < pad, lo, hi)  # the padding's own rows see nothing
    elif c["mask"] == "packed":  # causal inside each of the sequences of a row
        first = torch.rand(B, S, device="cuda", generator=g) < 8.0 / S
        lo = torch.where(first, i, 0).cummax(1).values
        hi = (i + 1).expand(B, S)
    elif c["mask"] == "windows":
        lo = (i // 64 * 64).expand(B, S)
        hi = (i // 64 * 64 + 64).clamp(max=S).expand(B, S)
    else:
        return None
    return torch.stack((lo, hi), -1).to(torch.int32).contiguous()


def _heads(B, S, H, D, dtype, g):
    """[B, H, S, D] as projections leave it: the tokens' memory is [B, S, H, D]."""
    return torch.randn(B, S, H, D, device="cuda", generator=g).to(dtype).transpose(1, 2)


def _quantise(x):
    scale = (x.float().abs().amax(-1) / F8_MAX).clamp(min=SCALE_MIN)
    return (x.float() / scale[..., None]).to(F8), scale


def prepare(case, seed):
    c, g = case, torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    s = {"case": c}
    if c["kind"] == "qknorm":
        B, S, Hq, Hkv, D = c["B"], c["S"], c["Hq"], c["Hkv"], c["D"]
        qkv = torch.randn(B, S, (Hq + 2 * Hkv) * D, device="cuda", generator=g).to(dt)  # the projection's result
        q, k, _ = qkv.split([Hq * D, Hkv * D, Hkv * D], -1)
        s["q"], s["k"] = q.view(B, S, Hq, D).transpose(1, 2), k.view(B, S, Hkv, D).transpose(1, 2)
        s["wq"], s["wk"] = ((1 + 0.2 * torch.randn(D, device="cuda", generator=g)).to(dt) for _ in range(2))
        t = torch.arange(S, device="cuda") + torch.randint(0, c["far"] + 1, (B, 1), device="cuda", generator=g)
        s["pos"] = torch.stack((t, t + torch.randint(0, 32, t.shape, device="cuda", generator=g), t + torch.randint(0, 32, t.shape, device="cuda", generator=g)))
        s["inv_freq"] = 1.0 / THETA ** (torch.arange(0, D, 2, device="cuda", dtype=torch.float32) / D)
        s["planes"] = torch.tensor(_planes(D, c["layout"]), device="cuda")
        if c["src"] == "table":  # what the program builds once a forward: cos and sin in bf16, side by side
            cos, sin = (x.to(torch.bfloat16).view(torch.int16).to(torch.int32) & 0xffff for x in _angles(s))
            s["table"] = (cos | sin << 16)[..., : D // 2 if c["layout"] == "hf" else D].reshape(B * S, -1).contiguous()
        if c["grad"]:
            s["gq"], s["gk"] = _heads(B, S, Hq, D, dt, g), _heads(B, S, Hkv, D, dt, g)
            for n in ("q", "k", "wq", "wk"):
                s[n] = s[n].detach().requires_grad_()
    elif c["kind"] == "attn":
        B, Sq, Sk, D = c["B"], c["Sq"], c["Sk"], c["D"]
        s["q"], s["k"], s["v"] = _heads(B, Sq, c["Hq"], D, dt, g), _heads(B, Sk, c["Hkv"], D, dt, g), _heads(B, Sk, c["Hkv"], D, dt, g)
        s["ranges"] = _key_ranges(c, g)
        if c["grad"]:
            s["do"] = _heads(B, Sq, c["Hq"], D, dt, g)
            for n in ("q", "k", "v"):
                s[n] = s[n].detach().requires_grad_()
    else:
        B, C, Hkv, D = c["B"], c["C"], c["Hkv"], c["D"]
        for n in ("k", "v"):
            s[n + "_cache"], s[n + "_scale"] = _quantise(torch.randn(B, Hkv, C, D, device="cuda", generator=g) * 2)
        if c["kind"] == "write":
            s["k"], s["v"] = _heads(B, c["S"], Hkv, D, dt, g), _heads(B, c["S"], Hkv, D, dt, g)
            s["start"] = torch.randint(0, C - c["S"] + 1, (B,), device="cuda", generator=g).to(torch.int32)
            s["lengths"] = torch.randint(c["S"] // 2, c["S"] + 1, (B,), device="cuda", generator=g).to(torch.int32) if c["ragged"] else None
        else:
            s["q"] = _heads(B, c["Sq"], c["Hq"], D, dt, g)
            s["lengths"] = torch.randint(c["shortest"], c["longest"] + 1, (B,), device="cuda", generator=g).to(torch.int32)
    return s


# ----------------------------------------------------------------------------- the plain forms
def _angles(s):
    """cos and sin [B, S, D] in 64 bits."""
    a = s["pos"].double()[..., None] * s["inv_freq"].double().repeat(2)
    a = torch.gather(a, 0, s["planes"].expand(1, *a.shape[1:]))[0]
    return a.cos(), a.sin()


def _cos_sin(s):
    c = s["case"]
    if c["src"] == "positions":
        return (x.float()[:, None] for x in _angles(s))
    t = s["table"].view(c["B"], 1, c["S"], -1)
    t = t.repeat(1, 1, 1, 2) if c["layout"] == "hf" else t
    return (t << 16).view(torch.float32), (t & -65536).view(torch.float32)


def _turn(x):
    lo, hi = x.chunk(2, -1)
    return torch.cat((-hi, lo), -1)


def _plain_qknorm(s):
    c = s["case"]
    cos, sin = _cos_sin(s)

    def forward(x, w):
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        n = x * r * w
        return n * cos + _turn(n) * sin, r

    def backward(x, w, r, gy):
        gn = gy * cos - _turn(gy * sin)
        xh, gw = x * r, gn * w
        return r * (gw - xh * (gw * xh).mean(-1, keepdim=True)), (gn * xh).sum((0, 1, 2))

    dt = DTYPES[c["dtype"]]
    q, k, wq, wk = (s[n].detach().float() for n in ("q", "k", "wq", "wk"))
    (yq, rq), (yk, rk) = forward(q, wq), forward(k, wk)
    out = {"q": yq.to(dt), "k": yk.to(dt)}
    if c["grad"]:
        (dq, dwq), (dk, dwk) = backward(q, wq, rq, s["gq"].float()), backward(k, wk, rk, s["gk"].float())
        out.update(dq=dq.to(dt), dk=dk.to(dt), dwq=dwq.to(dt), dwk=dwk.to(dt))
    return out


def _visible(s, Sq, Sk):
    """bool [B or 1, 1, Sq, Sk]: which keys each query sees."""
    c = s["case"]
    j, i = torch.arange(Sk, device="cuda"), torch.arange(Sq, device="cuda")[:, None]
    end = s["lengths"].view(-1, 1, 1, 1) if s.get("lengths") is not None else torch.full((1, 1, 1, 1), Sk, device="cuda")
    see = j < end
    if c.get("causal") or c.get("mask") == "causal":
        see = see & (j <= end - Sq + i)
    if s.get("ranges") is not None:
        r = s["ranges"][:, None, :, None]
        see = see & (j >= r[..., 0]) & (j < r[..., 1])
    return see


def _softmax(q, k, see):
    p = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(q.size(-1))).masked_fill_(~see, -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp_(min=-3e38)).exp_()
    return p.div_(p.sum(-1, keepdim=True).clamp_(min=1e-38))


def _plain_attn(s, k, v):
    c = s["case"]
    group, dt = c["Hq"] // c["Hkv"], DTYPES[c["dtype"]]
    q = s["q"].detach().float().contiguous()
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    p = _softmax(q, k, _visible(s, q.size(2), k.size(2)))
    out = {"out": torch.matmul(p, v).to(dt)}
    if c.get("grad"):
        do = s["do"].float().contiguous()
        dv = torch.matmul(p.transpose(-1, -2).contiguous(), do)
        ds = torch.matmul(do, v.transpose(-1, -2).contiguous())
        ds.sub_((ds * p).sum(-1, keepdim=True)).mul_(p).mul_(1 / math.sqrt(c["D"]))
        dq = torch.matmul(ds, k)
        dk = torch.matmul(ds.transpose(-1, -2).contiguous(), q)
        out.update(dq=dq.to(dt), dk=dk.unflatten(1, (c["Hkv"], group)).sum(2).to(dt), dv=dv.unflatten(1, (c["Hkv"], group)).sum(2).to(dt))
    return out


def _plain_write(s):
    c = s["case"]
    at = torch.arange(c["S"], device="cuda")
    if s["lengths"] is None:
        b, t = torch.meshgrid(torch.arange(c["B"], device="cuda"), at, indexing="ij")
        b, t = b.reshape(-1), t.reshape(-1)
    else:
        b, t = (at < s["lengths"][:, None]).nonzero(as_tuple=True)
    to = s["start"][b].long() + t
    codes, scale = _quantise(torch.stack((s["k"], s["v"])).transpose(2, 3)[:, b, t])
    s["k_cache"].view(torch.uint8)[b, :, to] = codes[0].view(torch.uint8)
    s["v_cache"].view(torch.uint8)[b, :, to] = codes[1].view(torch.uint8)
    s["k_scale"][b, :, to], s["v_scale"][b, :, to] = scale[0], scale[1]


def _cache(s):
    return {n: s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}


def run(state):
    s, c = state, state["case"]
    if own:
        return _own(s, c)
    if c["kind"] == "qknorm":
        return _plain_qknorm(s)
    if c["kind"] == "attn":
        return _plain_attn(s, s["k"].detach().float(), s["v"].detach().float())
    if c["kind"] == "write":
        _plain_write(s)
        return _cache(s)
    return _plain_attn(s, *(s[n + "_cache"].float() * s[n + "_scale"][..., None] for n in "kv"))


def _own(s, c):
    ops = _ops()
    if c["kind"] == "qknorm":
        if c["src"] == "table":
            q, k = ops.qk_norm_rope_from_table(s["q"], s["k"], s["wq"], s["wk"], s["table"], _section(c["D"]), eps=EPS, layout=c["layout"])
        else:
            q, k = ops.qk_norm_rope_from_positions(s["q"], s["k"], s["wq"], s["wk"], s["pos"], s["inv_freq"], _section(c["D"]), eps=EPS, layout=c["layout"])
        out = {"q": q.detach(), "k": k.detach()}
        if c["grad"]:
            out["dq"], out["dk"], out["dwq"], out["dwk"] = torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["gq"], s["gk"]))
        return out
    if c["kind"] == "attn":
        y = ops.attention(s["q"], s["k"], s["v"], key_ranges=s["ranges"], causal=c["mask"] == "causal")
        out = {"out": y.detach()}
        if c["grad"]:
            out["dq"], out["dk"], out["dv"] = torch.autograd.grad(y, (s["q"], s["k"], s["v"]), s["do"])
        return out
    if c["kind"] == "write":
        ops.kv_cache_write(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["start"], lengths=s["lengths"])
        return _cache(s)
    return {"out": ops.cached_attention(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], key_lengths=s["lengths"], causal=c["causal"])}


# ----------------------------------------------------------------------------- what a pass cannot do without
def _pairs(c):
    """(query, key) pairs of one head, as the mask lets them through on average, and the keys of a row that anyone sees."""
    if c["kind"] == "cached":
        keys = (c["shortest"] + c["longest"]) / 2
        return c["B"] * c["Sq"] * keys, keys
    Sq, Sk = c["Sq"], c["Sk"]
    if c["mask"] == "full":
        return c["B"] * Sq * Sk, Sk
    if c["mask"] == "causal":
        return c["B"] * (Sq * (Sk - Sq) + Sq * (Sq + 1) / 2), Sk
    if c["mask"] == "windows":
        return c["B"] * Sq * min(64, Sq), Sk
    if c["mask"] == "packed":  # about eight sequences of a row
        return c["B"] * Sq * max(1.0, Sq / 8), Sk
    act, pad = min(32, Sq - Sq // 4), Sq // 4 * 0.25  # (a quarter of the half of the rows that are padded, over all)
    return c["B"] * ((Sq - pad) * (Sq - pad + 1) / 2 + act * (act - 1) / 2), Sk


def work(case):
    c = case
    e, D = BYTES[c["dtype"]], c["D"]
    if c["kind"] == "qknorm":
        heads = c["B"] * c["S"] * (c["Hq"] + c["Hkv"]) * D
        tables = c["B"] * c["S"] * (24 if c["src"] == "positions" else 2 * D if c["layout"] == "hf" else 4 * D)
        # forward: q and k in and out; backward: they and the gradients in, the gradients out
        return {"bytes": heads * e * (5 if c["grad"] else 2) + tables * (2 if c["grad"] else 1), "flops": heads * (24 if c["grad"] else 8)}
    if c["kind"] == "write":
        n = c["B"] * c["S"] * (0.75 if c["ragged"] else 1.0) * c["Hkv"]
        return {"bytes": 2 * n * (D * e + D + 4), "flops": 4 * n * D}
    pairs, keys = _pairs(c)
    rows = c["B"] * c["Sq"] * c["Hq"] * D * e
    if c["kind"] == "cached":
        return {"bytes": 2 * rows + 2 * c["B"] * keys * c["Hkv"] * (D + 4), "flops": 4 * pairs * c["Hq"] * D}
    kv = c["B"] * keys * c["Hkv"] * D * e
    if c["grad"]:  # forward, and backward with its five products
        return {"bytes": (2 + 4) * rows + (2 + 4) * kv, "flops": 14 * pairs * c["Hq"] * D}
    return {"bytes": 2 * rows + 2 * kv, "flops": 4 * pairs * c["Hq"] * D}


# ----------------------------------------------------------------------------- in 64 bits, from the definitions
def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "write":
        return None  # codes and their scales are what they are
    if c["kind"] == "qknorm":
        B, S, D = c["B"], c["S"], c["D"]
        leaves = [s[n].detach().double().requires_grad_(c["grad"]) for n in ("q", "k", "wq", "wk")]
        freq = torch.cat((s["inv_freq"], s["inv_freq"])).double()
        if c["src"] == "table":
            t = s["table"].view(B, S, -1)
            pair = torch.stack((t & 0xffff, (t >> 16) & 0xffff)).to(torch.int32)
            pair = (pair << 16).view(torch.float32).double()
            pair = torch.cat((pair, pair), -1) if c["layout"] == "hf" else pair
        else:
            angle = torch.stack([s["pos"][p].double() * freq[d] for d, p in enumerate(_planes(D, c["layout"]))], -1)
            pair = torch.stack((torch.cos(angle), torch.sin(angle)))
        z = torch.complex(pair[0], pair[1])[:, None]  # one turn per channel; the halves of a head may turn by different angles

        def result(x, w):
            n = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * w
            a, b = n[..., : D // 2], n[..., D // 2:]
            return torch.cat((a * z.real[..., : D // 2] - b * z.imag[..., : D // 2], b * z.real[..., D // 2:] + a * z.imag[..., D // 2:]), -1)

        y = result(leaves[0], leaves[2]), result(leaves[1], leaves[3])
        out = {"q": y[0].detach(), "k": y[1].detach()}
        if c["grad"]:
            out["dq"], out["dk"], out["dwq"], out["dwk"] = torch.autograd.grad(y, leaves, (s["gq"].double(), s["gk"].double()))
        return out
    q = s["q"].detach().double()
    if c["kind"] == "cached":
        k, v = (s[n + "_cache"].double() * s[n + "_scale"].double().unsqueeze(-1) for n in "kv")
    else:
        k, v = s["k"].detach().double(), s["v"].detach().double()
    B, Hq, Sq, D = q.shape
    group, Sk = Hq // c["Hkv"], k.size(2)
    if B * Hq > 4096:
        return None
    out = {"out": torch.empty_like(q)}
    if c.get("grad"):
        out.update(dq=torch.empty_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
    key = torch.arange(Sk, device="cuda")
    for b in range(B):
        end = torch.tensor(Sk, device="cuda") if s.get("lengths") is None else s["lengths"][b]
        first, last = torch.zeros(Sq, device="cuda"), end.expand(Sq)
        if c.get("causal") or c.get("mask") == "causal":
            last = torch.minimum(last, end - Sq + 1 + torch.arange(Sq, device="cuda"))
        if s.get("ranges") is not None:
            first, last = s["ranges"][b, :, 0], torch.minimum(last, s["ranges"][b, :, 1])
        hidden = (key < first[:, None]) | (key >= last[:, None])
        some = ~hidden.all(1, keepdim=True)
        for h in range(Hq):
            kk, vv = k[b, h // group], v[b, h // group]
            score = (q[b, h] @ kk.t() / math.sqrt(D)).masked_fill(hidden, -math.inf)
            prob = torch.where(some, torch.exp(score - torch.logsumexp(score, 1, keepdim=True)), 0.0)
            out["out"][b, h] = prob @ vv
            if c.get("grad"):
                g = s["do"][b, h].double()
                slope = prob * (g @ vv.t() - (g * out["out"][b, h]).sum(1, keepdim=True)) / math.sqrt(D)
                out["dv"][b, h // group] += prob.t() @ g
                out["dq"][b, h] = slope @ kk
                out["dk"][b, h // group] += slope.t() @ q[b, h]
    return out
