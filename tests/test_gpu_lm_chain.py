"""The language-model operators together, as a model uses them: tokens -> embedding -> layer norm -> gated recurrence, forward
and backward; on side streams, in captured graphs, and against differences."""
import pytest
import torch
import torch.nn.functional as F

from hfuse_b200 import ops
from oracle import lm

pytestmark = pytest.mark.gpu


def _model(dev, V, D, kind, seed=41):
    g = torch.Generator(device=dev).manual_seed(seed)
    table = torch.randn(V, D, generator=g, device=dev).to(kind)
    wg, bg, wx, bx = ((1 + 0.2 * torch.randn(D, generator=g, device=dev)).to(kind) for _ in range(4))
    return table, wg, bg, wx, bx


def _step(ids, dh, table, wg, bg, wx, bx):
    """One training step of one layer: the gate and the value are two norms of the same embeddings."""
    scale = table.shape[1] ** 0.5 / 4
    e = ops.embedding(table, ids, scale)
    gate, mg, rg = ops.layer_norm(e, wg, bg)
    x, mx, rx = ops.layer_norm(e, wx, bx)
    h, last, states = ops.gated_recurrence(gate, x, None, True)
    dgate, dx, _ = ops.gated_recurrence_backward(gate, x, states, dh)
    de1, dwg, dbg = ops.layer_norm_backward(e, dgate, mg, rg, wg)
    de2, dwx, dbx = ops.layer_norm_backward(e, dx, mx, rx, wx)
    dtable = ops.embedding_backward(de1 + de2, ids, table.shape[0], scale)
    return h, last, dtable, dwg, dbg, dwx, dbx


def _reference(ids, dh, *params):
    leaves = [p.double().requires_grad_() for p in params]
    table, wg, bg, wx, bx = leaves
    e = F.embedding(ids, table) * (table.shape[1] ** 0.5 / 4)
    gate, x = F.layer_norm(e, e.shape[-1:], wg, bg), F.layer_norm(e, e.shape[-1:], wx, bx)
    h, out = torch.zeros_like(x[:, 0]), []
    for t in range(x.shape[1]):
        a = torch.sigmoid(gate[:, t])
        h = a * h + (1 - a) * x[:, t]
        out.append(h)
    out = torch.stack(out, 1)
    return (out.detach(), h.detach()) + torch.autograd.grad((out * dh.double()).sum(), leaves)


def test_training_step_in_full_precision(dev):
    """About ten operators in a row, each within some hundred half steps of its result's scale: 2^-24 * 2^10 of the
    largest value of each output."""
    params = _model(dev, 211, 96, torch.float32)
    ids = torch.randint(0, 211, (3, 300), generator=torch.Generator(device=dev).manual_seed(42), device=dev)
    dh = torch.randn(3, 300, 96, generator=torch.Generator(device=dev).manual_seed(43), device=dev)
    for got, want in zip(_step(ids, dh, *params), _reference(ids, dh, *params)):
        assert (got.double() - want).abs().max() <= 2.0 ** -14 * want.abs().max()


def test_training_step_in_half_precision(dev):
    """Four tensors on the way are rounded to bf16 (half a step is 2^-8) and gradients pass through them: five
    roundings of the norm of each output."""
    params = _model(dev, 400, 128, torch.bfloat16)
    ids = torch.randint(0, 400, (4, 270), generator=torch.Generator(device=dev).manual_seed(44), device=dev)
    dh = torch.randn(4, 270, 128, generator=torch.Generator(device=dev).manual_seed(45), device=dev).bfloat16()
    for got, want in zip(_step(ids, dh, *params), _reference(ids, dh, *params)):
        assert (got.double() - want).norm() <= 5 * 2.0 ** -8 * want.norm()


def test_generation_step_by_step_equals_the_whole_sequence(dev):
    table, wg, bg, wx, bx = _model(dev, 50, 64, torch.float32)
    ids = torch.randint(0, 50, (2, 40), generator=torch.Generator(device=dev).manual_seed(46), device=dev)

    def run(i, h):
        e = ops.embedding(table, i, 2.0)
        return ops.gated_recurrence(ops.layer_norm(e, wg, bg)[0], ops.layer_norm(e, wx, bx)[0], h)[:2]

    whole, last = run(ids, None)
    h, out = None, []
    for t in range(40):
        y, h = run(ids[:, t:t + 1].contiguous(), h)
        out.append(y)
    # the inputs have the same bits; the two scans may add in another order, 40 steps of at most 40 half steps each
    tol = 1600 * lm.U * whole.abs().max()
    assert (torch.cat(out, 1) - whole).abs().max() <= tol and (h - last).abs().max() <= tol


@pytest.mark.parametrize("steps", [60, 290, 700])
def test_captured_step_replays_on_new_data_beside_another_graph(dev, steps):
    params = _model(dev, 300, 72, torch.bfloat16)
    g = torch.Generator(device=dev).manual_seed(47)
    ids = [torch.randint(0, 300, (2, steps), generator=g, device=dev) for _ in range(2)]
    dh = [torch.randn(2, steps, 72, generator=g, device=dev).bfloat16() for _ in range(2)]
    want = [[t.clone() for t in _step(i, d, *params)] for i, d in zip(ids, dh)]
    other = [[t.clone() for t in _step(i.flip(0), d, *params)] for i, d in zip(ids, dh)]
    slots, graphs, outs, streams = [], [], [], []
    for k in range(2):
        slot = (torch.zeros_like(ids[0]), torch.zeros_like(dh[0]))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            _step(*slot, *params)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(_step(*slot, *params))
        slots.append(slot), graphs.append(graph), streams.append(s)
    for k in range(2):
        for slot, i in zip(slots, (ids[k], ids[k].flip(0))):
            slot[0].copy_(i), slot[1].copy_(dh[k])
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                for _ in range(3):
                    graph.replay()
        torch.cuda.synchronize()
        for got, ref in zip(outs, (want[k], other[k])):
            for a, b in zip(got, ref):
                assert torch.equal(a, b)


def test_two_streams_at_once_and_a_given_stream(dev):
    params = _model(dev, 300, 64, torch.float32)
    g = torch.Generator(device=dev).manual_seed(48)
    sets = [(torch.randint(0, 300, (2, 500), generator=g, device=dev), torch.randn(2, 500, 64, generator=g, device=dev)) for _ in range(2)]
    want = [[t.clone() for t in _step(*s, *params)] for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for s, data in zip(streams, sets):
            with torch.cuda.stream(s):
                got.append(_step(*data, *params))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
    e = ops.embedding(params[0], sets[0][0], 1.0, stream=streams[1])
    streams[1].synchronize()
    assert torch.equal(e, ops.embedding(params[0], sets[0][0], 1.0))


@pytest.mark.parametrize("which", ["layer_norm", "embedding", "recurrence"])
def test_gradients_against_differences_of_the_kernels(dev, which):
    """<gradient, v> against (f(p + s v) - f(p - s v)) / 2s of the forward kernels.  The difference is off by the
    roundings of f's two values over 2 s (each term of the sum by at most 2^10 U of itself) and by s^2 / 6 times the third
    derivative along v, of the order of the first for inputs and directions of size one: 40 of it is granted."""
    g = torch.Generator(device=dev).manual_seed(49)
    s = 2.0 ** -8

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    if which == "layer_norm":
        p, dy = (normal(9, 130), normal(130), normal(130)), normal(9, 130)
        f = lambda *q: ops.layer_norm(*q)[0]  # noqa: E731
        _, m, r = ops.layer_norm(*p)
        grads = ops.layer_norm_backward(p[0], dy, m, r, p[1])
    elif which == "embedding":
        ids = torch.randint(0, 40, (200,), generator=g, device=dev)
        p, dy = (normal(40, 33),), normal(200, 33)
        f = lambda t: ops.embedding(t, ids, 1.5)  # noqa: E731
        grads = (ops.embedding_backward(dy, ids, 40, 1.5),)
    else:
        p, dy = (normal(2, 300, 20), normal(2, 300, 20), normal(2, 20)), normal(2, 300, 20)
        f = lambda *q: ops.gated_recurrence(*q)[0]  # noqa: E731
        _, _, states = ops.gated_recurrence(*p, True)
        grads = ops.gated_recurrence_backward(p[0], p[1], states, dy)
    v = [normal(*t.shape) for t in p]
    up, down = f(*[a + s * b for a, b in zip(p, v)]).double(), f(*[a - s * b for a, b in zip(p, v)]).double()
    slope = ((up - down) * dy.double()).sum() / (2 * s)
    size = ((up.abs() + down.abs()) * dy.double().abs()).sum()
    want = sum((a.double() * b.double()).sum() for a, b in zip(grads, v))
    tol = 2.0 ** 10 * lm.U * size / (2 * s) + 40 * s * s / 6 * sum((a.double() * b.double()).abs().sum() for a, b in zip(grads, v))
    assert abs(slope - want) <= tol
