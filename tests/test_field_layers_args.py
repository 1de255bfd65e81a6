"""What the embedding, the layer norm and the dropout refuse, checked on the host before
any launch (no GPU needed)."""

import ctypes
import sys

import pytest
import torch

from mlx3d_amd import _lib
from mlx3d_amd.nn import Dropout, Embedding, LayerNorm, dropout, embedding, layer_norm


def look(index=torch.int64, shape=(5, 3), dtype=torch.float32, scale=1.0):
    return embedding(torch.zeros((4,), dtype=index), torch.zeros(shape, dtype=dtype), scale)


@pytest.mark.parametrize("wrong, words", [
    (dict(index=torch.int16), "int32 or int64"),
    (dict(index=torch.float32), "int32 or int64"),
    (dict(dtype=torch.float64), "float32, bfloat16 or float16"),
    (dict(shape=(5,)), r"\(V, C\)"),
    (dict(shape=(0, 3)), "at least 1"),
    (dict(shape=(5, 0)), "at least 1"),
    (dict(scale=float("nan")), "finite"),
    (dict(scale=float("inf")), "finite"),
    (dict(scale=1e39), "finite"),
    (dict(), "GPU only"),
], ids=str)
def test_embedding_refuses(wrong, words):
    with pytest.raises(ValueError, match=words):
        look(**wrong)


def norm(x=(4, 6), w=(6,), b=(6,), dtype=torch.float32, wtype=None, eps=1e-5):
    made = [None if s is None else torch.zeros(s, dtype=wtype or dtype) for s in (w, b)]
    return layer_norm(torch.zeros(x, dtype=dtype), *made, eps=eps)


@pytest.mark.parametrize("wrong, words", [
    (dict(dtype=torch.float64), "float32, bfloat16 or float16"),
    (dict(dtype=torch.int32), "float32, bfloat16 or float16"),
    (dict(x=()), r"\(\.\.\., C\)"),
    (dict(x=(4, 0), w=(0,), b=(0,)), "at least 1"),
    (dict(w=(5,)), "shape"),
    (dict(b=(1, 6)), "shape"),
    (dict(wtype=torch.float16), "type"),
    (dict(eps=0.0), "eps"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=1e-39), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(eps=float("inf")), "eps"),
    (dict(w=None, b=None), "GPU only"),
    (dict(), "GPU only"),
], ids=str)
def test_layer_norm_refuses(wrong, words):
    with pytest.raises(ValueError, match=words):
        norm(**wrong)


def drop(dtype=torch.float32, residual=None, rtype=None, p=0.5, seed=1, offset=0):
    r = None if residual is None else torch.zeros(residual, dtype=rtype or dtype)
    return dropout(torch.zeros((4, 6), dtype=dtype), p, seed, offset, r)


@pytest.mark.parametrize("wrong, words", [
    (dict(dtype=torch.float64), "float32, bfloat16 or float16"),
    (dict(residual=(6,)), "shape and type"),
    (dict(residual=(4, 6), rtype=torch.float16), "shape and type"),
    (dict(p=-0.1), r"\[0, 1\]"),
    (dict(p=1.1), r"\[0, 1\]"),
    (dict(p=float("nan")), r"\[0, 1\]"),
    (dict(seed=-1), "seed"),
    (dict(seed=1 << 64), "seed"),
    (dict(seed=1.5), "seed"),
    (dict(offset=-1), "offset"),
    (dict(offset=1 << 63), "offset"),
    (dict(offset=0.5), "offset"),
    (dict(offset=torch.zeros((2,), dtype=torch.int64)), "offset"),
    (dict(offset=torch.zeros((1,), dtype=torch.int32)), "offset"),
    (dict(offset=torch.zeros((1,), dtype=torch.int64)), "GPU only"),
    (dict(), "GPU only"),
], ids=str)
def test_dropout_refuses(wrong, words):
    with pytest.raises(ValueError, match=words):
        drop(**wrong)


def test_modules_refuse():
    with pytest.raises(ValueError, match="at least 1"):
        Embedding(0, 4, device="cpu")
    with pytest.raises(ValueError, match="scale"):
        Embedding(3, 4, scale=0.0, device="cpu")
    with pytest.raises(ValueError, match="at least 1"):
        LayerNorm(0, device="cpu")
    with pytest.raises(ValueError, match=r"\[0, 1\]"):
        Dropout(2.0, seed=0, device="cpu")
    with pytest.raises(ValueError, match="seed"):
        Dropout(0.5, seed=-1, device="cpu")
    with pytest.raises(ValueError, match="GPU only"):
        Embedding(3, 4, device="cpu")(torch.zeros((2,), dtype=torch.int64))
    with pytest.raises(ValueError, match="GPU only"):
        LayerNorm(4, device="cpu")(torch.zeros(3, 4))
    with pytest.raises(ValueError, match="GPU only"):
        Dropout(0.5, seed=1, device="cpu")(torch.zeros(3, 4))
    a, b = (Embedding(3, 4, device="cpu", seed=5).params["table"] for _ in range(2))
    assert torch.equal(a, b)


def test_missing_nodes_are_named(monkeypatch):
    """Without the native nodes the layers raise; there is no other path."""
    monkeypatch.setattr(_lib, "_autograd", None)
    monkeypatch.setitem(sys.modules, "mlx3d_amd._autograd", None)
    monkeypatch.delattr("mlx3d_amd._autograd", raising=False)
    with pytest.raises(ImportError, match="_autograd.so is missing"):
        _lib.autograd()


def test_the_nodes_hear_of_timers():
    from mlx3d_amd import profiling

    heard = []
    profiling.watch(heard.append)
    try:
        with profiling.StageTimer():
            with profiling.StageTimer():
                pass
    finally:
        profiling._watchers.remove(heard.append)
    assert heard == [False, True, True, True, False]
    assert _lib.autograd() is _lib.autograd()


BUF = (ctypes.c_char * 4096)()
P = ctypes.c_void_p((ctypes.addressof(BUF) + 255) // 256 * 256)  # never dereferenced
ODD = ctypes.c_void_p(P.value + 1)
BIG = 1 << 40


def swapped(good, changes):
    for at, bad in changes:
        args = list(good)
        args[at] = bad
        yield args


def test_the_lookup_entries_refuse():
    L = _lib.load()
    # dtype, count, rows, width
    for head, rc in (((3, 4, 5, 6), -1), ((0, -1, 5, 6), -1), ((0, 4, 0, 6), -1),
                     ((0, 4, 5, 0), -1), ((0, (1 << 30) + 1, 5, 6), -4),
                     ((0, 4, (1 << 30) + 1, 6), -4), ((0, 4, 5, (1 << 20) + 1), -4)):
        assert L.gsx_embed_bwd_workspace_bytes(*head) == rc
        assert L.gsx_embed_fwd(*head, P, 0, P, 1 << 21, 1.0, P, None) == rc
        assert L.gsx_embed_bwd(*head, P, 0, P, 1 << 21, 1.0, P, P, BIG, None) == rc
    head = (0, 4, 5, 6)
    good = [P, 0, P, 6, 1.0, P]
    for args in swapped(good, ((0, None), (0, ODD), (1, 2), (2, None), (2, ODD), (3, 5),
                               (4, float("nan")), (4, float("inf")), (5, None), (5, ODD))):
        assert L.gsx_embed_fwd(*head, *args, None) == -1
        assert L.gsx_embed_bwd(*head, *args, P, BIG, None) == -1
    need = L.gsx_embed_bwd_workspace_bytes(*head)
    assert need > 0
    assert L.gsx_embed_bwd(*head, *good, P, need - 1, None) == -3
    assert L.gsx_embed_bwd(*head, *good, None, need, None) == -3
    assert L.gsx_embed_bwd(*head, *good, ctypes.c_void_p(P.value + 8), need, None) == -1
    # int64 indices are aligned to theirs
    assert L.gsx_embed_fwd(*head, ctypes.c_void_p(P.value + 4), 1, *good[2:], None) == -1


def test_the_norm_entries_refuse():
    L = _lib.load()
    for head, rc in (((3, 4, 6), -1), ((0, -1, 6), -1), ((0, 4, 0), -1),
                     ((0, (1 << 30) + 1, 6), -4), ((0, 4, (1 << 20) + 1), -4)):
        assert L.gsx_layer_norm_bwd_workspace_bytes(*head) == rc
        assert L.gsx_layer_norm_fwd(*head, P, 1 << 21, P, P, 1e-5, P, None) == rc
        assert L.gsx_layer_norm_bwd(*head, P, 1 << 21, P, P, 1 << 21, 1e-5, P, P, P, P, BIG,
                                    None) == rc
    head = (0, 4, 6)
    for args in swapped([P, 6, P, P, 1e-5, P], ((0, None), (0, ODD), (1, 5), (2, ODD), (3, ODD),
                                                (4, 0.0), (4, float("nan")), (4, float("inf")),
                                                (5, None), (5, ODD))):
        assert L.gsx_layer_norm_fwd(*head, *args, None) == -1
    good = [P, 6, P, P, 6, 1e-5, P, P, P]
    for args in swapped(good, ((0, None), (0, ODD), (1, 5), (2, ODD), (3, None), (3, ODD), (4, 5),
                               (5, 0.0), (6, ODD), (7, ODD), (8, ODD))):
        assert L.gsx_layer_norm_bwd(*head, *args, P, BIG, None) == -1
    for width in (6, 9000):
        need = L.gsx_layer_norm_bwd_workspace_bytes(0, 4, width)
        wide = [P, width, P, P, width, 1e-5, P, P, P]
        assert need > 0
        assert L.gsx_layer_norm_bwd(0, 4, width, *wide, P, need - 1, None) == -3
        assert L.gsx_layer_norm_bwd(0, 4, width, *wide, None, need, None) == -3
    assert L.gsx_layer_norm_bwd(*head, *good, ctypes.c_void_p(P.value + 8), BIG, None) == -1


def test_the_dropout_entry_refuses():
    L = _lib.load()
    good = [0, 24, 0.5, 1, 0, None, P, P, P]
    for args in swapped(good, ((0, 3), (1, -1), (2, -0.5), (2, 1.5), (2, float("nan")), (4, -1),
                               (5, ctypes.c_void_p(P.value + 4)), (6, None), (6, ODD), (7, ODD),
                               (8, None), (8, ODD))):
        assert L.gsx_dropout(*args, None) == -1
    assert L.gsx_dropout(0, (1 << 34) + 1, *good[2:], None) == -4
