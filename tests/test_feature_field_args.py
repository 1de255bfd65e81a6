"""What the feature field's operators refuse, checked on the host before any
launch (no GPU needed)."""

import ctypes

import pytest
import torch

from mlx3d_amd import _lib
from mlx3d_amd.losses import distillation_loss, distillation_value_and_grad
from mlx3d_amd.nn import GatedFeedForward, gated_feed_forward


def block(x=(4, 8), wg=(16, 8), wu=(16, 8), wd=(3, 16), dtype=torch.float32, wtype=None,
          act="silu"):
    w = [torch.zeros(s, dtype=wtype or dtype) for s in (wg, wu, wd)]
    return gated_feed_forward(torch.zeros(x, dtype=dtype), *w, activation=act)


@pytest.mark.parametrize("wrong, words", [
    (dict(act="relu"), "activation"),
    (dict(dtype=torch.float64), "float32, bfloat16 or float16"),
    (dict(wtype=torch.float16), "one type"),
    (dict(x=(4, 9)), "hidden, d_in"),
    (dict(wu=(15, 8)), "hidden, d_in"),
    (dict(wg=(16,), wu=(16,)), "hidden, d_in"),
    (dict(wd=(3, 15)), "d_out, hidden"),
    (dict(wd=(0, 16)), "at least 1"),
    (dict(x=(4, 0), wg=(16, 0), wu=(16, 0)), "at least 1"),
    (dict(), "GPU only"),
], ids=str)
def test_block_refuses(wrong, words):
    with pytest.raises(ValueError, match=words):
        block(**wrong)


def test_module_refuses():
    with pytest.raises(ValueError, match="activation"):
        GatedFeedForward(4, 8, 2, activation="tanh", device="cpu")
    with pytest.raises(ValueError, match="at least 1"):
        GatedFeedForward(4, 0, 2, device="cpu")
    m = GatedFeedForward(4, 8, 2, device="cpu", seed=3)
    same = GatedFeedForward(4, 8, 2, device="cpu", seed=3)
    assert all(torch.equal(m.params[k], same.params[k]) for k in m.params)
    with pytest.raises(ValueError, match="GPU only"):
        m(torch.zeros(3, 4))


def told(logits=(4, 9), values=(4, 2), index=None, dtype=torch.float32, vtype=torch.float32,
         itype=torch.int64, call=distillation_loss, **how):
    return call(torch.zeros(logits, dtype=dtype), torch.zeros(values, dtype=vtype),
                torch.zeros(index or values, dtype=itype), **how)


@pytest.mark.parametrize("wrong, words", [
    (dict(dtype=torch.float64), "float32, bfloat16 or float16"),
    (dict(vtype=torch.int32), "floating point"),
    (dict(itype=torch.int16), "int32 or int64"),
    (dict(index=(4, 3)), "shape"),
    (dict(values=(5, 2)), "leading"),
    (dict(values=(2,)), "shape"),
    (dict(values=(4, 10)), "between 1 and"),
    (dict(values=(4, 0)), "between 1 and"),
    (dict(logits=(4, 400), values=(4, 257)), "between 1 and"),
    (dict(temperature=0.0), "temperature"),
    (dict(temperature=-1.0), "temperature"),
    (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=float("inf")), "temperature"),
    (dict(teacher="probs"), "teacher"),
    (dict(reduction="batch"), "reduction"),
    (dict(call=distillation_value_and_grad, reduction="none"), "scalar"),
    (dict(), "GPU only"),
], ids=lambda v: str({k: getattr(w, "__name__", w) for k, w in v.items()})
    if isinstance(v, dict) else v)
def test_distillation_refuses(wrong, words):
    with pytest.raises(ValueError, match=words):
        told(**wrong)


def test_c_entries_refuse_before_a_launch():
    L = _lib.load()
    buf = (ctypes.c_char * 4096)()
    p = ctypes.c_void_p((ctypes.addressof(buf) + 255) // 256 * 256)  # never dereferenced
    odd = ctypes.c_void_p(p.value + 1)
    big = 1 << 40
    # dtype, act, rows, widths
    for head, rc in (((3, 0, 4, 8, 8, 8), -1), ((0, 3, 4, 8, 8, 8), -1), ((0, 0, -1, 8, 8, 8), -1),
                     ((0, 0, 4, 0, 8, 8), -1), ((0, 0, 4, 8, 8, 0), -1),
                     ((0, 0, (1 << 30) + 1, 8, 8, 8), -4), ((0, 0, 4, 8, (1 << 20) + 1, 8), -4)):
        assert L.gsx_ffn_fwd_workspace_bytes(*head) == rc
        assert L.gsx_ffn_bwd_workspace_bytes(*head) == rc
        assert L.gsx_ffn_fwd(*head, p, 8, p, p, p, p, p, big, None) == rc
        assert L.gsx_ffn_bwd(*head, p, 8, p, p, p, p, 8, p, p, p, p, p, big, None) == rc
    head = (0, 0, 4, 8, 8, 8)
    need = L.gsx_ffn_fwd_workspace_bytes(*head)
    assert L.gsx_ffn_fwd(*head, p, 8, p, p, p, p, p, need - 1, None) in (-3, -1)
    assert L.gsx_ffn_fwd(*head, None, 8, p, p, p, p, p, big, None) == -1
    assert L.gsx_ffn_fwd(*head, p, 7, p, p, p, p, p, big, None) == -1
    assert L.gsx_ffn_fwd(*head, odd, 8, p, p, p, p, p, big, None) == -1
    assert L.gsx_ffn_bwd(*head, p, 8, p, p, p, p, 7, p, p, p, p, p, big, None) == -1
    assert L.gsx_ffn_bwd(*head, p, 8, p, p, p, p, 8, p, p, None, p, p, big, None) == -1
    assert L.gsx_ffn_bwd(*head, p, 8, p, p, p, p, 8, p, p, p, p, p, 16, None) == -3
    # dtype, rows, vocab, top
    for head, rc in (((3, 4, 9, 2), -1), ((0, -1, 9, 2), -1), ((0, 4, 0, 1), -1),
                     ((0, 4, 9, 0), -1), ((0, 4, 9, 10), -1), ((0, 4, 999, 257), -4),
                     ((0, 1 << 30, 9, 2), -4)):
        assert L.gsx_distil_workspace_bytes(*head) == rc
        assert L.gsx_distil_fwd(*head, p, 9999, p, p, 0, 1.0, 0, 2, p, p, big, None) == rc
    head = (0, 4, 9, 2)
    need = L.gsx_distil_workspace_bytes(*head)
    good = [p, 9, p, p, 0, 1.0, 0, 2]
    for at, bad in ((0, None), (0, odd), (1, 8), (2, None), (3, odd), (4, 2), (5, 0.0), (6, 2),
                    (7, 3)):
        args = list(good)
        args[at] = bad
        assert L.gsx_distil_fwd(*head, *args, p, p, big, None) == -1
        assert L.gsx_distil_bwd(*head, *args, p, p, p, big, None) == -1
        assert L.gsx_distil_fwd_bwd(*head, *args, 1.0, p, p, p, big, None) == -1
    assert L.gsx_distil_fwd(*head, *good, p, p, need - 1, None) == -3
    assert L.gsx_distil_fwd(*head, *good, None, p, big, None) == -1
    assert L.gsx_distil_bwd(*head, *good, None, p, p, big, None) == -1
    assert L.gsx_distil_fwd_bwd(*head, *good[:7], 0, 1.0, p, p, p, big, None) == -1


def test_more_segments_than_a_launch_holds_are_refused():
    """Rows over 8192 bytes take a workgroup of 256 threads for each 16 KB."""
    L = _lib.load()
    for dtype, rows, vocab, rc in ((1, 1 << 24, 4097, -4), (0, 1 << 24, 2049, -4),
                                   (1, (1 << 24) // 3 + 1, 16385, -4), (1, 1 << 24, 4096, 0),
                                   (1, (1 << 24) - 1, 4097, 0), (1, (1 << 24) // 3, 16385, 0)):
        need = L.gsx_distil_workspace_bytes(dtype, rows, vocab, 2)
        assert need == rc if rc else need > 0
