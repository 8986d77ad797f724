"""What the attention, cache and norm entry points refuse on the host, before any launch (no GPU needed), and the masks that
attention_key_ranges builds."""

import pytest
import torch

from wallx_mi355 import _lib, native
from wallx_mi355.fusions import ops

BF16, F16, F32 = _lib.WX_BF16, _lib.WX_F16, _lib.WX_F32
ST = _lib.i64x3((4096, 128, 256))


def _fwd(p, batch=1, nq=2, nkv=1, sq=4, sk=4, d=128, qs=ST, ks=ST, vs=ST, scale=0.1, dtype=BF16, q=None, ranges=None):
    lib = _lib.load()
    return lib.wx_attention_fwd(p if q is None else q, p, p, p, None, None, ranges, None, 0, batch, nq, nkv, sq, sk, d, qs, ks, vs, scale, dtype, None, 0, None)


@pytest.fixture()
def buf():
    t = torch.zeros(64)
    return t, (t.data_ptr() + 15) // 16 * 16  # never dereferenced: the calls fail on the host


def test_attention_forward_refuses(buf):
    _, p = buf
    lib = _lib.load()
    assert _fwd(p, d=96) == -2 and b"64, 80 or 128" in lib.wx_last_error_string()
    assert _fwd(p, dtype=F32) == -2
    assert _fwd(p, nq=3, nkv=2) == -1 and b"no multiple" in lib.wx_last_error_string()
    assert _fwd(p, nq=2, nkv=0) == -1
    assert _fwd(p, batch=-1) == -1 and _fwd(p, sk=-1) == -1
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert _fwd(p, scale=scale) == -1 and b"scale" in lib.wx_last_error_string()
    assert _fwd(None) == -1 and b"null pointer" in lib.wx_last_error_string()
    assert _fwd(p, q=p + 8) == -1 and b"16-byte" in lib.wx_last_error_string()
    assert _fwd(p, ranges=p + 4) == -1 and b"8-byte" in lib.wx_last_error_string()
    assert _fwd(p, ks=_lib.i64x3((4096, 128, 252))) == -2 and _fwd(p, qs=_lib.i64x3((4096, 128, -256))) == -2
    assert _fwd(p, ks=_lib.i64x3((0, 0, 2 ** 25))) == -2 and b"too large" in lib.wx_last_error_string()
    assert _fwd(p, sq=2 ** 30) == -2 and _fwd(p, sk=2 ** 30) == -2
    assert _fwd(p, qs=None) == -1
    # one query over many keys is split: its sums need room
    assert lib.wx_attention_workspace_bytes(1, 8, 1, 1, 32768, 128) > 0
    assert _fwd(p, nq=8, sq=1, sk=32768) == -3 and b"workspace" in lib.wx_last_error_string()
    # nothing to do
    assert _fwd(None, batch=0) == 0 and _fwd(None, sq=0) == 0
    assert lib.wx_attention_workspace_bytes(16, 16, 2, 912, 912, 128) == 0


def test_attention_backward_refuses(buf):
    _, p = buf
    lib = _lib.load()

    def bwd(nq=2, nkv=1, sq=4, sk=4, d=128, dtype=BF16, gs=ST, x=p, ws=None, n=0):
        return lib.wx_attention_bwd(x, x, x, x, x, None, x, x, x, x, None, None, 0, 1, nq, nkv, sq, sk, d, ST, ST, ST, gs, 0.1, dtype, ws, n, None)

    assert bwd(d=72) == -2 and bwd(dtype=F32) == -2 and bwd(nq=3, nkv=2) == -1
    assert bwd(x=None) == -1 and bwd(gs=None) == -1 and bwd(gs=_lib.i64x3((4096, 129, 256))) == -2
    assert bwd(gs=_lib.i64x3((4096, 2 ** 30, 256))) == -2 and b"too large" in lib.wx_last_error_string()
    assert bwd(nq=1025) == -2 and b"1024" in lib.wx_last_error_string()
    assert bwd() == -3 and b"workspace" in lib.wx_last_error_string()
    assert bwd(ws=p, n=lib.wx_attention_bwd_workspace_bytes(1, 2, 1, 4, 4, 128) - 1) == -3
    assert lib.wx_attention_bwd(*([None] * 12), 0, 0, 2, 1, 4, 4, 128, ST, ST, ST, ST, 0.1, BF16, None, 0, None) == 0


def test_cache_refuses(buf):
    _, p = buf
    lib = _lib.load()

    def write(k=p, cache=p, d=128, dtype=BF16, st=ST, batch=1, cap=8, start=p):
        return lib.wx_kv_cache_write(k, k, cache, cache, p, p, start, None, batch, 1, 4, cap, d, st, st, dtype, None)

    assert write(d=96) == -2 and write(dtype=F32) == -2 and write(batch=-1) == -1
    assert write(k=None) == -1 and write(start=None) == -1 and write(st=None) == -1
    assert write(cache=p + 8) == -1 and write(st=_lib.i64x3((4096, 128, 4))) == -2
    assert write(batch=0) == 0 and write(cap=0) == 0
    args = (None, None, 0, 1, 2, 1, 4, 8, 128, ST)
    assert lib.wx_cached_attention(p, p, p, p, None, p, *args, 0.1, BF16, None, 0, None) == -1
    assert lib.wx_cached_attention(p, p + 8, p, p, p, p, *args, 0.1, BF16, None, 0, None) == -1
    assert lib.wx_cached_attention(p, p, p, p, p, p, *args, 0.1, F32, None, 0, None) == -2


def test_norm_refuses(buf):
    _, p = buf
    lib = _lib.load()
    sec = _lib.i32x3((16, 24, 24))

    def norm(q=p, w=p, freq=p, d=128, dtype=BF16, s=sec, layout=0, eps=1e-6, st=ST, batch=1):
        return lib.wx_qk_norm_rope(q, p, w, p, eps, p, freq, p, p, batch, 4, 2, 1, d, st, st, s, layout, dtype, None)

    assert norm(d=80, s=_lib.i32x3((10, 15, 15))) == -2 and b"power of two" in lib.wx_last_error_string()
    assert norm(s=_lib.i32x3((16, 24, 25))) == -1
    assert norm(q=None) == -1 and norm(w=None) == -1 and norm(st=None) == -1 and norm(s=None) == -1
    assert norm(q=p + 8) == -1 and norm(w=p + 8) == -1 and norm(st=_lib.i64x3((4096, 128, 4))) == -2
    assert norm(eps=-1.0) == -1 and norm(eps=float("nan")) == -1 and norm(dtype=7) == -2 and norm(layout=3) == -1
    assert norm(freq=None, dtype=F16) == -2 and b"bf16" in lib.wx_last_error_string()
    assert norm(batch=0) == 0
    assert lib.wx_qk_norm_rope_bwd(p, p, p, p, p, p, 1e-6, p, p, p, p, p, p, 1, 4, 2, 1, 128, ST, ST, ST, ST, sec, 0, BF16, None, 0, None) == -3
    assert lib.wx_qk_norm_rope_bwd(p, None, p, p, p, p, 1e-6, p, p, p, p, None, None, 1, 4, 2, 1, 128, ST, ST, ST, ST, sec, 0, BF16, None, 0, None) == -1


def test_ops_refuse_cpu_tensors():
    q, w = torch.zeros(1, 2, 3, 64), torch.zeros(64)
    with pytest.raises(RuntimeError, match="on the device: CPU"):
        ops.attention(q, q, q)
    with pytest.raises(RuntimeError, match="on the device: CPU"):
        ops.cached_attention(q, q, q, w, w)
    with pytest.raises(RuntimeError, match="on the device: CPU"):
        ops.kv_cache_write(q, q, q, q, w, w, w)
    with pytest.raises(RuntimeError, match="on the device: CPU"):
        ops.qk_norm_rope_from_table(q, q, w, w, w, [8, 8, 16])
    with pytest.raises(RuntimeError, match="on the device: CPU"):
        ops.qk_norm_rope_from_positions(q, q, w, w, w, w, [8, 8, 16])


@pytest.mark.parametrize("padded", [None, "left", "right", "both", "all"])
def test_key_ranges(padded):
    B, S = 4, 23
    types = torch.zeros(B, S, dtype=torch.bool)
    types[0, 15:21], types[1, 3:6], types[2, 22] = True, True, True
    keep = torch.ones(B, S, dtype=torch.bool)
    if padded in ("left", "both"):
        keep[0, :4], keep[1, :4] = False, False
    if padded in ("right", "both"):
        keep[0, 18:], keep[2, 20:] = False, False
    if padded == "all":
        keep[3] = False
    r = ops.attention_key_ranges(types, None if padded is None else keep.long())
    act = types & keep
    see = (torch.ones(S, S, dtype=torch.bool).tril() | (act[:, :, None] & act[:, None, :])) & keep[:, None, :] & keep[:, :, None]
    j = torch.arange(S)
    assert r.shape == (B, S, 2) and r.dtype == torch.int32
    assert torch.equal((j >= r[..., :1]) & (j < r[..., 1:]), see)


def test_key_ranges_in_checked_mode():
    types = torch.zeros(2, 9, dtype=torch.int64)
    types[1, 2], types[1, 5] = 1, 1
    keep = torch.ones(2, 9, dtype=torch.int64)
    ops.attention_key_ranges(types, keep)
    native.set_checked(True)
    try:
        with pytest.raises(ValueError, match="action tokens"):
            ops.attention_key_ranges(types, keep)
        keep[0, 4] = 0
        with pytest.raises(ValueError, match="unpadded tokens"):
            ops.attention_key_ranges(types * 0, keep)
        ops.attention_key_ranges(types * 0)
    finally:
        native.set_checked(False)
    with pytest.raises(RuntimeError, match="batch, seq"):
        ops.attention_key_ranges(types[0])
    assert ops.attention_key_ranges(types[:, :0]).shape == (2, 0, 2)
