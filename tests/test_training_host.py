"""Refusals of the norm, rotation and gradient entry points that need no GPU: the C ABI checks its
arguments before any launch (the stand-in pointers are never dereferenced), the Python layer refuses
CPU tensors."""
import pytest
import torch

import mod_dit_amd as md
from mod_dit_amd import _lib, ops

P = 16  # a non-null, 16-byte aligned stand-in pointer


def _rope(q=P, k=P, sizes=(1, 2, 64, 64, 64), strides=(0, 0, 0), dtype=0, norm=1, across=0, eps=1e-6, w=(P, P),
          b=(None, None), w_dtype=2, tables=(P, P), tab=(0, 64), tab_dim=64, off=0, n=64):
    s = _lib.strides3(*strides)
    return _lib.load().moddit_qk_norm_rope(q, k, P, P, *sizes, s, s, s, s, dtype, norm, across, eps, *w, *b, w_dtype,
                                           *tables, _lib.strides2(*tab), tab_dim, off, n, 1, None)


def _rope_bwd(sums=(None,) * 4, norm=1, w=(P, P), ws=None, floats=0, sizes=(1, 2, 64, 64, 64)):
    s = _lib.strides3(0, 0, 0)
    return _lib.load().moddit_qk_norm_rope_bwd(P, P, P, P, P, P, *sums, *sizes, s, s, s, s, s, s, 0, norm, 0, 1e-6, *w,
                                               2, None, None, _lib.strides2(0, 0), 0, 0, 0, 1, ws, floats, None)


@pytest.mark.parametrize("kw,rc,word", [
    (dict(sizes=(1, 2, 64, 64, 96)), _lib.MODDIT_EUNSUPPORTED, b"head_dim"),
    (dict(sizes=(1, -1, 64, 64, 64)), _lib.MODDIT_EINVAL, b"negative"),
    (dict(dtype=2), _lib.MODDIT_EUNSUPPORTED, b"dtype"),
    (dict(norm=3), _lib.MODDIT_EINVAL, b"norm"),
    (dict(norm=0), _lib.MODDIT_EINVAL, b"need a norm"),
    (dict(norm=0, w=(None, None), across=1), _lib.MODDIT_EINVAL, b"need a norm"),
    (dict(eps=-1.0), _lib.MODDIT_EINVAL, b"eps"),
    (dict(eps=float("nan")), _lib.MODDIT_EINVAL, b"eps"),
    (dict(w_dtype=7), _lib.MODDIT_EINVAL, b"weight dtype"),
    (dict(sizes=(1, 129, 64, 64, 64), across=1), _lib.MODDIT_EUNSUPPORTED, b"8192"),
    (dict(off=-1), _lib.MODDIT_EINVAL, b"offset"),
    (dict(off=1), _lib.MODDIT_EINVAL, b"exceed"),
    (dict(sizes=(1, 2, 64, 63, 64)), _lib.MODDIT_EINVAL, b"exceed"),
    (dict(tables=(None, P)), _lib.MODDIT_EINVAL, b"tables missing"),
    (dict(tab_dim=48), _lib.MODDIT_EINVAL, b"head_dim / 2"),
    (dict(tab=(0, -64)), _lib.MODDIT_EINVAL, b"table strides"),
    (dict(strides=(0, 0, 4)), _lib.MODDIT_EINVAL, b"multiples of 8"),
    (dict(strides=(0, -8, 0)), _lib.MODDIT_EINVAL, b"multiples of 8"),
    (dict(q=None), _lib.MODDIT_EINVAL, b"null"),
    (dict(k=P + 8), _lib.MODDIT_EINVAL, b"aligned"),
])
def test_qk_norm_rope_refuses(kw, rc, word):
    assert _rope(**kw) == rc
    assert word in _lib.load().moddit_last_error()


def test_qk_norm_rope_of_nothing_is_done_without_a_launch():
    assert _rope(q=None, k=None, sizes=(0, 2, 64, 64, 64)) == _lib.MODDIT_OK
    assert _rope(q=None, k=None, sizes=(1, 2, 0, 0, 64), n=0) == _lib.MODDIT_OK


def test_qk_norm_rope_bwd_refuses():
    lib = _lib.load()
    assert _rope_bwd(sums=(P, None, None, None), norm=0, w=(None, None)) == _lib.MODDIT_EINVAL
    assert b"need a norm" in lib.moddit_last_error()
    need = lib.moddit_qk_norm_rope_bwd_workspace_floats(1, 2, 64, 64, 64, 0)
    assert need > 0 and lib.moddit_qk_norm_rope_bwd_workspace_floats(1, 2, 64, 64, 80, 0) == 0
    assert _rope_bwd(sums=(P, None, None, None)) == _lib.MODDIT_EINVAL
    assert b"workspace" in lib.moddit_last_error()
    assert _rope_bwd(sizes=(1, 2, -1, 64, 64)) == _lib.MODDIT_EINVAL
    assert _rope_bwd(sizes=(0, 2, 64, 64, 64)) == _lib.MODDIT_OK


def _bwd(sparse=False, q=P, sizes=(1, 2, 64, 64, 64), stride=64, scale=0.125, dtype=0, lists=None, origin=0, ws=P,
         nbytes=1 << 30):
    s = _lib.strides3(0, 0, stride)
    args = (q, P, P, P, P, P, None, P, P, P, *sizes, *([s] * 8), scale, dtype)
    if not sparse:
        return _lib.load().moddit_flash_bwd(*args, ws, nbytes, None)
    lists = (P, P, 1, 1, P, P, 1, 2) if lists is None else lists
    return _lib.load().moddit_block_sparse_bwd(*args, *lists, origin, ws, nbytes, None)


@pytest.mark.parametrize("kw,rc,word", [
    (dict(sizes=(1, 2, 64, 64, 96)), _lib.MODDIT_EUNSUPPORTED, b"head_dim"),
    (dict(sizes=(1, 2, -1, 64, 64)), _lib.MODDIT_EINVAL, b"negative"),
    (dict(sizes=(2, 40000, 64, 64, 64)), _lib.MODDIT_EINVAL, b"65535"),
    (dict(dtype=2), _lib.MODDIT_EUNSUPPORTED, b"dtype"),
    (dict(scale=0.0), _lib.MODDIT_EINVAL, b"softmax_scale"),
    (dict(scale=float("inf")), _lib.MODDIT_EINVAL, b"softmax_scale"),
    (dict(stride=60), _lib.MODDIT_EINVAL, b"multiples of 8"),
    (dict(q=None), _lib.MODDIT_EINVAL, b"null"),
    (dict(q=P + 2), _lib.MODDIT_EINVAL, b"aligned"),
    (dict(ws=None), _lib.MODDIT_EINVAL, b"workspace"),
    (dict(ws=P + 4), _lib.MODDIT_EINVAL, b"workspace"),
    (dict(nbytes=16), _lib.MODDIT_EINVAL, b"workspace"),
    (dict(stride=0), _lib.MODDIT_EINVAL, b"at least head_dim"),
    (dict(stride=1 << 25), _lib.MODDIT_EUNSUPPORTED, b"2 GiB"),
    (dict(sparse=True, lists=(None, P, 1, 1, P, P, 1, 2)), _lib.MODDIT_EINVAL, b"counts"),
    (dict(sparse=True, lists=(P, P, 1, 1, None, P, 1, 2)), _lib.MODDIT_EINVAL, b"lists missing"),
    (dict(sparse=True, lists=(P, P, 2, 1, P, P, 1, 2)), _lib.MODDIT_EINVAL, b"n_qtiles"),
    (dict(sparse=True, lists=(P, P, 1, 1, P, P, 2, 2)), _lib.MODDIT_EINVAL, b"n_ktiles"),
    (dict(sparse=True, lists=(P, P, 1, 0, P, P, 1, 2)), _lib.MODDIT_EINVAL, b"cap"),
    (dict(sparse=True, origin=-64), _lib.MODDIT_EINVAL, b"grid_origin"),
    (dict(sparse=True, origin=1), _lib.MODDIT_EINVAL, b"grid_origin"),
])
def test_attention_bwd_refuses(kw, rc, word):
    assert _bwd(**kw) == rc
    assert word in _lib.load().moddit_last_error()


def test_attention_bwd_of_nothing_is_done_without_a_launch():
    assert _bwd(q=None, sizes=(1, 0, 64, 64, 64)) == _lib.MODDIT_OK
    assert _bwd(q=None, sizes=(1, 2, 0, 0, 64), ws=None) == _lib.MODDIT_OK
    assert _bwd(sparse=True, q=None, sizes=(1, 2, 0, 0, 64), lists=(None, None, 0, 0) * 2, ws=None) == _lib.MODDIT_OK


def test_transpose_tiles_refuses():
    lib = _lib.load()
    assert lib.moddit_transpose_tiles(P, P, 1, 2, 4, P, P, 2, 3, None) == _lib.MODDIT_EINVAL
    assert b"key_cap" in lib.moddit_last_error()
    assert lib.moddit_transpose_tiles(P, P, 1, 6145, 4, P, P, 2, 12290, None) == _lib.MODDIT_EUNSUPPORTED
    assert lib.moddit_transpose_tiles(None, P, 1, 2, 4, P, P, 2, 4, None) == _lib.MODDIT_EINVAL
    assert lib.moddit_transpose_tiles(None, None, 0, 2, 4, None, None, 2, 4, None) == _lib.MODDIT_OK


def test_python_layer_refuses_cpu_tensors_and_table_gradients():
    q = torch.zeros(1, 2, 8, 64, dtype=torch.bfloat16)
    lse = torch.zeros(1, 2, 8)
    tiles = ops.TileList(torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, 1, 1, dtype=torch.int32), 64, False)
    for call in (lambda: ops.qk_norm_rope(q, q), lambda: ops.qk_norm_rope_bwd(q, q, q, q),
                 lambda: ops.flash_bwd(q, q, q, q, lse, q), lambda: ops.block_sparse_bwd(q, q, q, q, lse, q, tiles),
                 lambda: ops.transpose_tiles(tiles, 8), lambda: md.flash_attention(q, q, q)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    cos = torch.zeros(8, 64, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        md.qk_norm_rope(q, q, cos=cos, sin=cos)
