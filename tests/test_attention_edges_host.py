"""The attention entry points at the edges of what they take, on the host (no GPU needed: nothing is launched)."""

import torch

from wallx_mi355 import _lib

BF16 = _lib.WX_BF16
ST = _lib.i64x3((4096, 128, 256))


def test_backward_without_query_heads():
    """The gradients of keys that no head reads are written as well, and take their workspace; without keys there is nothing to do."""
    lib = _lib.load()
    t = torch.zeros(64)
    p = (t.data_ptr() + 15) // 16 * 16  # never dereferenced: the calls end on the host

    def bwd(sk=4, nkv=1, k=p, ws=None, n=0):
        return lib.wx_attention_bwd(None, k, k, None, None, None, None, None, k, k, None, None, 0, 1, 0, nkv, 4, sk, 128, ST, ST, ST, ST, 0.1, BF16, ws, n, None)

    need = lib.wx_attention_bwd_workspace_bytes(1, 0, 1, 4, 4, 128)
    assert need > 0 and bwd() == -3 and b"workspace" in lib.wx_last_error_string()
    assert bwd(ws=p, n=need - 1) == -3 and bwd(k=None, ws=p, n=need) == -1
    assert bwd(nkv=0) == 0 and lib.wx_attention_bwd_workspace_bytes(1, 0, 0, 4, 4, 128) == 0


def test_more_threads_than_a_launch_holds():
    """2^32 threads and more along a grid's x are refused in front of the first launch (the runtime starts them modulo 2^32)."""
    lib = _lib.load()
    t = torch.zeros(64)
    p = (t.data_ptr() + 15) // 16 * 16
    sec = _lib.i32x3((16, 24, 24))

    def write(batch, heads=1, seq=1):
        return lib.wx_kv_cache_write(p, p, p, p, p, p, p, None, batch, heads, seq, 8, 128, ST, ST, BF16, None)

    def fwd(batch, sq=1, ws=None, n=0):
        return lib.wx_attention_fwd(p, p, p, p, None, None, None, None, 0, batch, 1, 1, sq, 1, 128, ST, ST, ST, 0.1, BF16, ws, n, None)

    def bwd(batch, sq=1, sk=1):
        return lib.wx_attention_bwd(p, p, p, p, p, None, p, p, p, p, None, None, 0, batch, 1, 1, sq, sk, 128, ST, ST, ST, ST, 0.1, BF16, p, 2 ** 62, None)

    def norm(batch):
        return lib.wx_qk_norm_rope(p, p, p, p, 1e-6, p, p, p, p, batch, 1, 1, 1, 128, ST, ST, sec, 0, BF16, None)

    for call in (lambda: write(2 ** 24), lambda: write(1, 2, 2 ** 27), lambda: fwd(2 ** 24), lambda: fwd(2 ** 22, 512), lambda: bwd(2 ** 24), lambda: bwd(2 ** 22),
                 lambda: bwd(2 ** 21, 1, 512), lambda: norm(2 ** 28)):
        assert call() == -2 and b"too many" in lib.wx_last_error_string()
    cached = lib.wx_cached_attention(p, p, p, p, p, p, None, None, 0, 2 ** 24, 1, 1, 1, 1, 128, ST, 0.1, BF16, None, 0, None)
    assert cached == -2 and b"too many" in lib.wx_last_error_string()
    assert lib.wx_mrope_table(p, p, 2 ** 26, 1, 128, sec, 0, p, None) == -2 and b"too many" in lib.wx_last_error_string()
