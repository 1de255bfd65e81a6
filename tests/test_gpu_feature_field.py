"""The decoder and its loss as they are used: the example's training, graph
capture, the widths and row counts at which the block changes kernels, and rows
whose result may not depend on how many others there are."""

import importlib.util
import os

import pytest
import torch

from mlx3d_amd.losses import distillation_loss, distillation_value_and_grad
from mlx3d_amd.nn import gated_feed_forward
from test_gpu_distil import inputs as told
from test_gpu_feed_forward import ACTS, TYPES, check, formulas, inputs, outputs

pytestmark = pytest.mark.gpu

DEV = "cuda"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_example_learns_its_labels():
    spec = importlib.util.spec_from_file_location(
        "distil_feature_field", os.path.join(ROOT, "examples", "distil_feature_field.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, same = example.train(steps=80, n=1500, size=96, verbose=False)
    assert losses[-1] < 0.25 * losses[0], (losses[0], losses[-1])
    assert same > 0.8, same


# hidden groups of one to four pairs, several groups, widths on both sides of
# each kernel's limit, row pitches below eight, workgroups with many tiles
SIZES = [(500, 20, 300, 40), (333, 40, 200, 20), (100, 3, 600, 5), (2100, 7, 700, 300),
         (31, 32, 128, 64), (33, 32, 96, 64), (1000, 64, 64, 64), (30000, 8, 40, 12),
         (900, 100, 513, 30), (450, 128, 512, 32), (450, 129, 64, 32), (450, 32, 64, 129),
         (450, 33, 64, 33), (450, 64, 160, 65), (450, 32, 512, 128), (450, 32, 513, 128),
         (700, 6, 530, 6), (513, 300, 40, 7), (260, 32, 2000, 16), (8, 128, 300, 256),
         (4096, 2, 33, 2)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_block_where_kernels_change(size, dtype):
    act = ACTS[(sum(size) + 1) % 3]
    t = inputs(*size, dtype, seed=sum(size))
    check(outputs(*t, act), *formulas(*t, act), dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("widths", [(27, 100, 21), (32, 128, 64), (200, 90, 150)], ids=str)
def test_a_row_is_the_same_among_others(widths, dtype):
    """Outputs and row gradients keep their bits whichever rows stand beside them."""
    x, wg, wu, wd, dy = inputs(700, *widths, dtype, seed=2)
    whole = outputs(x, wg, wu, wd, dy, "silu")
    for first, n in ((0, 1), (5, 40), (131, 300), (699, 1)):
        part = outputs(x[first:first + n], wg, wu, wd, dy[first:first + n], "silu")
        for k in ("y", "dx"):
            assert torch.equal(part[k], whole[k][first:first + n]), (k, first, n)


@pytest.mark.parametrize("teacher", ["logits", "log_probs"])
@pytest.mark.parametrize("rows, vocab, top", [(9000, 21, 3), (5000, 150, 8), (1200, 1500, 20)])
def test_a_rows_loss_is_the_same_among_others(rows, vocab, top, teacher):
    for dtype in TYPES:
        logits, values, index = told(rows, vocab, top, dtype, teacher, seed=3)
        how = dict(teacher=teacher, temperature=1.5)
        each = distillation_loss(logits, values, index, reduction="none", **how)
        total, grad = distillation_value_and_grad(logits, values, index, reduction="sum", **how)
        assert abs(float(total) - float(each.double().sum())) <= 1e-6 * float(each.double().sum())
        for first, n in ((0, 1), (3, 50), (rows // 2, 130), (rows - 1, 1)):
            part = slice(first, first + n)
            e = distillation_loss(logits[part], values[part], index[part], reduction="none", **how)
            t, g = distillation_value_and_grad(logits[part], values[part], index[part],
                                               reduction="sum", **how)
            assert torch.equal(e, each[part]) and torch.equal(g, grad[part])
        mean, g = distillation_value_and_grad(logits, values, index, **how)
        active = ((index >= 0) & (index < vocab) & (values != -float("inf"))).any(1).sum()
        assert abs(float(mean) * int(active) - float(total)) <= 1e-6 * float(total)


@pytest.mark.parametrize("rows, vocab", [(40, 21), (4000, 150), (6, 9000)])
def test_graph_replays(rows, vocab):
    """Captured, and replayed between eager work: every replay against eager."""
    logits, values, index = told(rows, vocab, 4, torch.float32, "logits", seed=4)
    x, wg, wu, wd, _ = inputs(rows, 24, 72, vocab if vocab < 200 else 40, torch.float32, seed=5)

    def work():
        y = gated_feed_forward(x, wg, wu, wd)
        return (y, *distillation_value_and_grad(logits, values, index))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    g = torch.Generator().manual_seed(0)
    for _ in range(4):
        x.copy_(torch.randn(x.shape, generator=g))
        logits.copy_(torch.randn(logits.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, work()):
            assert torch.equal(a, b)
