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
