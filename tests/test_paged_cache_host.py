"""What the paged cache's entry points refuse on the host, before any launch (no GPU needed)."""

import pytest
import torch

from wallx_mi355 import _lib
from wallx_mi355.fusions import ops

BF16, F32 = _lib.WX_BF16, _lib.WX_F32
ST = _lib.i64x3((4096, 128, 256))


@pytest.fixture()
def p():
    t = torch.zeros(64)
    yield (t.data_ptr() + 15) // 16 * 16  # never dereferenced: the calls fail on the host


def test_resize_refuses(p):
    lib = _lib.load()

    def resize(x=p, requests=4, width=8, capacity=32, ps=16, tokens=64, count=p, slots=p):
        return lib.wx_paged_kv_resize(x, x, x, x, count, x, x, x, slots, slots, requests, width, capacity, ps, tokens, None)

    assert resize(requests=-1) == -1 and resize(width=-1) == -1 and resize(capacity=-1) == -1 and resize(tokens=-1) == -1
    assert resize(ps=0) == -1 and resize(ps=-4) == -1 and b"page_size" in lib.wx_last_error_string()
    assert resize(requests=4097) == -2 and b"4096 requests" in lib.wx_last_error_string()
    assert resize(width=2 ** 26) == -2 and b"tokens to a request" in lib.wx_last_error_string()
    assert resize(capacity=2 ** 27) == -2 and b"slots" in lib.wx_last_error_string()
    assert resize(requests=4096, width=2 ** 16) == -2 and resize(tokens=2 ** 30) == -2
    assert resize(x=None) == -1 and resize(count=None) == -1 and resize(slots=None) == -1 and b"null pointer" in lib.wx_last_error_string()
    assert resize(slots=p + 8) == -1 and b"16-byte" in lib.wx_last_error_string()


def test_write_refuses(p):
    lib = _lib.load()

    def write(x=p, pages=p, scales=(p, p), slots=p, batch=1, nkv=2, seq=3, n=4, ps=16, d=128, ks=ST, vs=ST, dtype=BF16):
        return lib.wx_paged_kv_write(x, x, pages, pages, *scales, slots, batch, nkv, seq, n, ps, d, ks, vs, dtype, None)

    assert write(batch=-1) == -1 and write(nkv=-1) == -1 and write(seq=-1) == -1 and write(n=-1) == -1 and write(ps=0) == -1
    assert write(d=96) == -2 and write(dtype=F32) == -2 and write(ks=None) == -1 and write(ks=_lib.i64x3((0, 4, 8))) == -2
    assert write(scales=(p, None)) == -1 and write(scales=(None, p)) == -1 and b"neither" in lib.wx_last_error_string()
    assert write(x=None) == -1 and write(pages=None) == -1 and write(slots=None) == -1 and write(pages=p + 8) == -1
    assert write(n=2 ** 27) == -2 and write(seq=2 ** 30) == -2 and write(batch=2 ** 20, seq=2 ** 10) == -2 and write(seq=2 ** 29) == -2
    for nothing in (dict(batch=0), dict(nkv=0), dict(seq=0), dict(n=0)):
        assert write(x=None, **nothing) == 0


def test_attention_refuses(p):
    lib = _lib.load()

    def attend(q=p, pages=p, scales=(p, p), table=p, lengths=p, starts=p, batch=1, nq=4, nkv=2, seq=3, requests=2, width=4, n=8, ps=16, d=128, st=ST, scale=0.1,
               dtype=BF16):
        return lib.wx_paged_attention(q, pages, pages, *scales, q, table, lengths, starts, 1, batch, nq, nkv, seq, requests, width, n, ps, d, st, scale, dtype, None, 0,
                                      None)

    for name in ("batch", "nq", "nkv", "seq", "requests", "width", "n"):
        assert attend(**{name: -1}) == -1, name
    assert attend(ps=0) == -1 and attend(d=72) == -2 and attend(dtype=F32) == -2 and attend(nq=3) == -1 and attend(nkv=0) == -1
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert attend(scale=scale) == -1
    assert attend(scales=(p, None)) == -1 and attend(st=None) == -1 and attend(st=_lib.i64x3((0, 129, 256))) == -2 and attend(st=_lib.i64x3((0, -128, 256))) == -2
    assert attend(starts=None) == -1 and b"row of q" in lib.wx_last_error_string()
    assert attend(q=None) == -1 and attend(pages=None) == -1 and attend(table=None) == -1 and attend(lengths=None) == -1 and attend(pages=p + 8) == -1
    assert attend(nq=4098) == -2 and attend(seq=2 ** 29) == -2 and attend(batch=2 ** 20, seq=2 ** 10) == -2 and attend(width=2 ** 27) == -2 and attend(n=2 ** 28) == -2
    assert attend(q=None, seq=0) == 0 and attend(q=None, batch=0) == 0 and attend(q=None, nq=0, nkv=0) == 0


def test_ops_refuse_the_cpu():
    x = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16)
    cache = ops.paged_kv_cache(4, 2, 16, 64, "cpu")
    state = ops.paged_kv_tables(2, 2, 4, "cpu")
    assert [tuple(t.shape) for t in cache] == [(4, 2, 16, 64)] * 2 + [(4, 2, 16)] * 2 and ops.paged_kv_cache(4, 2, 16, 64, "cpu", torch.float16)[2:] == (None, None)
    assert state[2].tolist() == [3, 2, 1, 0] and state[3].tolist() == [4] and state[1].tolist() == [[-1, -1]] * 2
    with pytest.raises(RuntimeError, match="CPU"):
        ops.paged_kv_resize(state[0], state[0], *state[1:], 16, 4)
    with pytest.raises(RuntimeError, match="CPU"):
        ops.paged_kv_write(x, x, *cache, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CPU"):
        ops.paged_attention(x, *cache, state[1], state[0])
