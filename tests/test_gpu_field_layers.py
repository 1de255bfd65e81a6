"""Embedding, layer norm and dropout as they are used: together around the decoder,
captured into graphs, under checkpointing, on several streams, and rows whose results may
not depend on how many others there are."""

import importlib.util
import os
import threading

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from mlx3d_amd import _lib
from mlx3d_amd.cameras import Camera
from mlx3d_amd.losses import distillation_loss
from mlx3d_amd.nn import (Dropout, Embedding, GatedFeedForward, LayerNorm, dropout, embedding,
                          layer_norm)
from mlx3d_amd.splatting import render_gaussian_features

pytestmark = pytest.mark.gpu

DEV = "cuda"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = (torch.float32, torch.bfloat16, torch.float16)


class Decoder:
    """A token's row of a table, a pre-norm residual block with dropout, and the logits."""

    def __init__(self, rows=300, width=24, classes=11, dtype=torch.float32):
        self.table = Embedding(rows, width, scale=2.0, dtype=dtype, seed=1)
        self.norm = LayerNorm(width, dtype=dtype)
        self.block = GatedFeedForward(width, 40, width, dtype=dtype, seed=2)
        self.drop = Dropout(0.25, seed=5)
        self.out = GatedFeedForward(width, 32, classes, dtype=dtype, seed=3)
        self.leaves = [p for part in (self.table, self.norm, self.block, self.out)
                       for p in part.params.values()]

    def __call__(self, tokens):
        h = self.table(tokens)
        h = self.drop(self.block(self.norm(h)), h)
        return self.out(h)


def targets(count, classes=11, top=3, seed=0):
    g = torch.Generator().manual_seed(seed)
    index = torch.stack([torch.randperm(classes, generator=g)[:top] for _ in range(count)])
    return torch.randn((count, top), generator=g).to(DEV), index.to(DEV)


def tokens_of(count, rows=300, seed=0):
    g = torch.Generator().manual_seed(seed)
    k = (rows * torch.rand((count,), generator=g) ** 2).long().clamp_(max=rows - 1)
    k[::17] = -1
    return k.to(DEV)


def plain(decoder, tokens, values, index):
    """The same in float64 elementary operations, with the dropout's own mask."""
    leaf = [p.detach().double().requires_grad_(True) for p in decoder.leaves]
    table, w, b, g1, u1, d1, g2, u2, d2 = leaf
    there = tokens >= 0
    h = torch.where(there[:, None], table[torch.where(there, tokens, 0)] * 2.0, 0.0)
    m = h.mean(dim=1, keepdim=True)
    n = (h - m) / (((h - m) ** 2).mean(dim=1, keepdim=True) + 1e-5).sqrt() * w + b
    act = torch.nn.functional.silu
    f = (act(n @ g1.T) * (n @ u1.T)) @ d1.T
    kept = dropout(torch.ones_like(f, dtype=torch.float32), 0.25, 5, int(decoder.drop.step)) != 0
    h = h + torch.where(kept, f / 0.75, 0.0)
    logits = (act(h @ g2.T) * (h @ u2.T)) @ d2.T
    p = torch.softmax(values.double(), dim=1)
    log_q = torch.log_softmax(logits, dim=1).gather(1, index)
    loss = (p * (p.log() - log_q)).sum(dim=1).mean()
    return loss, torch.autograd.grad(loss, leaf)


@pytest.mark.parametrize("count", (7, 500, 6000))
def test_a_step_of_all_of_them(count):
    """Loss and every gradient against float64: each operator's float32 sums are within
    1e-5 of theirs in the mean (their own tests), and five follow each other."""
    decoder, tokens = Decoder(), tokens_of(count)
    values, index = targets(count)
    for step in range(3):
        loss = distillation_loss(decoder(tokens), values, index)
        got = torch.autograd.grad(loss, decoder.leaves)
        want_loss, want = plain(decoder, tokens, values, index)
        assert abs(float(loss.detach() - want_loss.detach())) <= 5e-5 * float(want_loss.detach())
        for a, b in zip(got, want):
            assert float((a.double() - b).norm()) <= 5e-5 * float(b.norm())
        decoder.drop.advance()


@pytest.mark.parametrize("dtype", TYPES[1:], ids=str)
def test_a_step_in_16_bits(dtype):
    """Each of the chain's ten tensors and ten gradients is rounded once: at most twenty
    roundings of random sign, each to half a step, times the block's and the norm's own
    amplification of a few."""
    decoder, tokens = Decoder(dtype=dtype), tokens_of(3000)
    values, index = targets(3000)
    loss = distillation_loss(decoder(tokens), values, index, reduction="sum")
    got = torch.autograd.grad(loss, decoder.leaves)
    _, want = plain(decoder, tokens, values, index)
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    for a, b in zip(got, want):
        assert a.dtype == dtype
        assert float((a.double() / 3000 - b).norm()) <= 20 * half * float(b.norm())


def test_codes_rendered_and_decoded():
    """Gaussians that share a codebook, rendered, normalised and decoded: the table's
    gradient is the features' own, summed by code."""
    g = torch.Generator().manual_seed(0)
    n, codes = 500, 40
    means, quats = torch.randn((n, 3), generator=g) * 0.6, torch.randn((n, 4), generator=g)
    scales = torch.exp(torch.randn((n, 3), generator=g) * 0.3 - 2.4)
    scene = [t.to(DEV) for t in (means, quats, scales, torch.full((n,), 0.8))]
    camera = Camera.look_at(eye=(0, 0.3, -3.5), width=80, height=56, fov=45.0)
    table, norm = Embedding(codes, 16, seed=4), LayerNorm(16)
    block = GatedFeedForward(16, 48, 9, seed=5)
    code = torch.randint(-1, codes, (n,), generator=g).to(DEV)
    values, index = targets(56 * 80, classes=9)
    values, index = values.view(56, 80, 3), index.view(56, 80, 3)

    def loss_of(features):
        seen = render_gaussian_features(camera, *scene, features)["features"]
        return distillation_loss(block(norm(seen)), values, index)

    features = table(code)
    (of_table, of_features) = torch.autograd.grad(loss_of(features),
                                                  [table.params["table"], features])
    want = torch.zeros((codes, 16), dtype=torch.float64, device=DEV)
    there = code >= 0
    want.index_add_(0, code[there].long(), of_features[there].double())
    # a chain of at most n float32 additions a row
    size = torch.zeros_like(want).index_add_(0, code[there].long(),
                                             of_features[there].double().abs())
    assert bool(((of_table.double() - want).abs() <= (n + 1) * 2.0 ** -24 * size).all())
    assert float(of_table.norm()) > 0


def test_the_example_with_a_codebook():
    """It runs, and a step's gradients are those of the same step in plain operations
    behind the render (in float32: within what sums over some thousand pixels lose)."""
    spec = importlib.util.spec_from_file_location(
        "distil_feature_field", os.path.join(ROOT, "examples", "distil_feature_field.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, same = example.train(steps=6, n=800, size=64, verbose=False, codes=48)
    assert len(losses) == 6 and all(v == v and v < float("inf") for v in losses)
    assert 0.0 <= same <= 1.0
    means, *scene = example.scene(800)[:4]
    book = example.Codebook(means, 48)
    camera = example.cameras(1, 64)[0]
    leaves = [p for part in book.parts for p in part.values()]
    table, weight, bias = leaves

    def render(features):
        return render_gaussian_features(camera, means, *scene, features)["features"]

    rows = book.rows(render(book.features()))
    dy = torch.randn(rows.shape, generator=torch.Generator().manual_seed(2)).to(DEV)
    got = torch.autograd.grad(rows, leaves, dy)
    x = render(table[book.code])
    m = x.mean(dim=-1, keepdim=True)
    h = (x - m) / (((x - m) ** 2).mean(dim=-1, keepdim=True) + 1e-3).sqrt()
    kept = dropout(torch.ones_like(h), 0.1, 4, 0) != 0
    want = torch.autograd.grad(torch.where(kept, (h * weight + bias) / 0.9, 0.0), leaves, dy)
    for a, b in zip(got, want):
        assert float((a - b).norm()) <= 5e-5 * float(b.norm())


def test_captured_steps():
    """Forward, gradients and the dropout's next step in one graph: every replay against
    the same step in eager mode, between replays of another graph of its own inputs."""
    held = []
    for seed, count in ((0, 5000), (1, 20_000)):
        decoder, tokens = Decoder(), tokens_of(count, seed=seed)
        values, index = targets(count, seed=seed)

        def work(decoder=decoder, tokens=tokens, values=values, index=index):
            loss = distillation_loss(decoder(tokens), values, index)
            grads = torch.autograd.grad(loss, decoder.leaves)
            decoder.drop.advance()
            return (loss.detach(), *grads)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = work()
        held.append((graph, out, work, decoder, tokens))
    for _ in range(3):
        for graph, out, work, decoder, tokens in held:
            tokens.copy_(tokens.roll(3))
            graph.replay()
        torch.cuda.synchronize()
        for graph, out, work, decoder, tokens in held:
            decoder.drop.step -= 1
            for a, b in zip(out, work()):
                assert torch.equal(a, b)


def test_two_streams_at_once():
    """Calls on two streams, of other sizes, that may run beside each other."""
    jobs = []
    for seed, count in ((0, 30_000), (1, 9000)):
        g = torch.Generator().manual_seed(seed)
        x = torch.randn((count, 48), generator=g).to(DEV).requires_grad_(True)
        w = torch.randn((48,), generator=g).to(DEV).requires_grad_(True)
        table = torch.randn((300, 48), generator=g).to(DEV).requires_grad_(True)
        jobs.append((x, w, table, tokens_of(count, seed=seed)))

    def work(x, w, table, tokens):
        y = dropout(layer_norm(x, w), 0.5, 9, 4, embedding(tokens, table))
        return (y.detach(), *torch.autograd.grad(y, [x, w, table], x.detach()))

    want = [work(*j) for j in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, j in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(work(*j))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("width", (3, 5, 8, 27, 40, 100, 200, 257, 700, 1365, 5000, 9000))
def test_a_row_is_the_same_among_others(width, dtype):
    g = torch.Generator().manual_seed(width)
    x, dy = (torch.randn((90, width), generator=g).to(dtype).to(DEV) for _ in range(2))
    w, b = (torch.randn((width,), generator=g).to(dtype).to(DEV) for _ in range(2))

    def both(x, dy):
        x = x.detach().requires_grad_(True)
        y = layer_norm(x, w, b)
        return y.detach(), torch.autograd.grad(y, x, dy)[0]

    whole = both(x, dy)
    for first, n in ((0, 1), (3, 40), (89, 1)):
        part = slice(first, first + n)
        assert all(torch.equal(p, q[part]) for p, q in zip(both(x[part], dy[part]), whole))


def ops():
    g = torch.Generator().manual_seed(0)
    x, w, b, r = (torch.randn(s, generator=g).to(DEV).requires_grad_(True)
                  for s in ((50, 8), (8,), (8,), (50, 8)))
    k = torch.randint(0, 50, (70,), generator=g).to(DEV)
    step = torch.full((1,), 3, dtype=torch.int64, device=DEV)
    return [(lambda x, w, b: layer_norm(x, w, b), (x, w, b)),
            (lambda x: layer_norm(x), (x,)),
            (lambda x: embedding(k, x, 2.0), (x,)),
            (lambda x, r: dropout(x, 0.5, 1, 2, r), (x, r)),
            (lambda x: dropout(x, 0.5, 1, step), (x,))]


@pytest.mark.parametrize("which", range(5))
def test_a_penalty_on_the_gradient_is_refused(which):
    call, leaves = ops()[which]
    y = call(*leaves).square().sum()
    grads = torch.autograd.grad(y, leaves, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (leaves[0].square().sum() + grads[0].square().sum()).backward()


@pytest.mark.parametrize("which", range(5))
@pytest.mark.parametrize("create_graph", (False, True))
def test_gradients_through_a_checkpoint(which, create_graph):
    call, leaves = ops()[which]
    dy = torch.randn(call(*leaves).shape, generator=torch.Generator().manual_seed(1)).to(DEV)
    want = torch.autograd.grad(call(*leaves), leaves, dy)
    got = torch.autograd.grad(checkpoint(call, *leaves, use_reentrant=False), leaves, dy,
                              create_graph=create_graph)
    for a, b in zip(got, want):
        assert torch.equal(a.detach(), b)


@pytest.mark.parametrize("which", range(5))
@pytest.mark.parametrize("mode", (torch.no_grad, torch.inference_mode))
def test_without_a_graph(which, mode):
    call, leaves = ops()[which]
    want = call(*leaves).detach()
    with mode():
        y = call(*(t.detach() for t in leaves))
        assert not y.requires_grad and torch.equal(y, want)


def test_threads_at_once():
    """Forward and gradient from four threads, each on a stream of its own."""
    call, leaves = ops()[0]
    dy = torch.randn((50, 8), generator=torch.Generator().manual_seed(1)).to(DEV)
    want = torch.autograd.grad(call(*leaves), leaves, dy)
    torch.cuda.synchronize()
    wrong = []

    def work():
        mine = [t.detach().clone().requires_grad_(True) for t in leaves]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                got = torch.autograd.grad(call(*mine), mine, dy)
            torch.cuda.current_stream().synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want)):
                wrong.append(threading.get_ident())

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_inputs_changed_before_the_gradient_are_noticed():
    call, (x,) = ops()[2]
    k = torch.zeros((4,), dtype=torch.int64, device=DEV)
    y = embedding(k, x)
    k += 1
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    z = x.detach().clone().requires_grad_(True)
    h = z * 1.0
    y = layer_norm(h)
    h.detach().add_(0)  # shares the storage, and its version
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


def test_a_timer_sees_the_stages():
    from mlx3d_amd.profiling import StageTimer

    with StageTimer() as timer:
        for call, leaves in ops():
            call(*leaves).sum().backward()
    for name in ("layer_norm_fwd", "layer_norm_bwd", "embed_fwd", "embed_bwd", "dropout"):
        assert timer.mean_ms(name) > 0


def test_errors_of_the_entry_points_reach_the_caller():
    x = torch.zeros((4, 4), device=DEV)
    with pytest.raises(_lib.GsxError, match="gsx_dropout failed"):
        _lib.autograd().dropout(x, None, 1.5, 1, 0, None)
    with pytest.raises(_lib.GsxError, match="gsx_layer_norm_fwd failed"):
        _lib.autograd().layer_norm(x, None, None, 0.0)
