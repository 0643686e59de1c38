"""The 64-bit definitions of the language-model operators: gradients against differences and torch's own operators."""
import pytest
import torch
import torch.nn.functional as F

from oracle import lm


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _difference(f, inputs, seed):
    """(central difference of f along a random direction, that direction)"""
    g = _gen(seed)
    v = [torch.randn(t.shape, generator=g, dtype=torch.float64) for t in inputs]
    h = 1e-6
    up = f(*[t + h * d for t, d in zip(inputs, v)])
    down = f(*[t - h * d for t, d in zip(inputs, v)])
    return (up - down) / (2 * h), v


def test_layer_norm_and_its_gradient():
    g = _gen(1)
    x, w, b, dy = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((5, 7), (7,), (7,), (5, 7)))
    y, mean, invstd = lm.layer_norm(x, w, b, 1e-5)
    torch.testing.assert_close(y, F.layer_norm(x, (7,), w, b, 1e-5), rtol=1e-12, atol=1e-12)
    grads = lm.layer_norm_backward(x, dy, mean, invstd, w)
    slope, v = _difference(lambda *t: (lm.layer_norm(*t, 1e-5)[0] * dy).sum(), (x, w, b), 2)
    assert abs(slope - sum((a * d).sum() for a, d in zip(grads, v))) < 1e-7 * (1 + abs(slope))


def test_embedding_and_its_gradient():
    g = _gen(3)
    table = torch.randn(6, 4, generator=g, dtype=torch.float64)
    ids = torch.tensor([[1, 5, 1], [0, -1, 6]])
    dy = torch.randn(2, 3, 4, generator=g, dtype=torch.float64)
    out = lm.embedding(table, ids, 2.5)
    assert (out[1, 1] == 0).all() and (out[1, 2] == 0).all() and torch.equal(out[0, 0], table[1] * 2.5)
    grad = lm.embedding_backward(dy, ids, 6, 2.5)
    slope, v = _difference(lambda t: (lm.embedding(t, ids, 2.5) * dy).sum(), (table,), 4)
    assert abs(slope - (grad * v[0]).sum()) < 1e-7 * (1 + abs(slope))
    assert (lm.embedding_backward(dy, ids, 6, 2.5, padding_id=1)[1] == 0).all()


@pytest.mark.parametrize("start", [False, True])
def test_gated_recurrence_and_its_gradient(start):
    g = _gen(5)
    gate, x, dy = (torch.randn(2, 9, 3, generator=g, dtype=torch.float64) for _ in range(3))
    h0, dl = (torch.randn(2, 3, generator=g, dtype=torch.float64) for _ in range(2))
    h0 = h0 if start else torch.zeros_like(h0)
    dg, dx, dh0, _ = lm.gated_recurrence_backward(gate, x, h0, dy, dl)

    def loss(gate, x, h0):
        h, _, last = lm.gated_recurrence(gate, x, h0)
        return (h * dy).sum() + (last * dl).sum()

    slope, v = _difference(loss, (gate, x, h0), 6)
    assert abs(slope - sum((a * d).sum() for a, d in zip((dg, dx, dh0), v))) < 1e-7 * (1 + abs(slope))


def test_gates_of_infinity_start_afresh_and_hold():
    x = torch.tensor([[[1.0], [2.0], [3.0], [4.0]]])
    gate = torch.tensor([[[0.0], [float("-inf")], [float("inf")], [0.0]]])
    h = lm.gated_recurrence(gate, x, torch.tensor([[5.0]]))[0].flatten().tolist()
    assert h == [3.0, 2.0, 2.0, 3.0]
