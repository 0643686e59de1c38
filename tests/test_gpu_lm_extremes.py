"""The language-model operators at the ends of their inputs' ranges, against the 64-bit definitions."""
import pytest
import torch

from hfuse_b200 import ops
from oracle import lm
from test_gpu_lm import TYPES, _check_rec, _gen, _ids, api  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- gates in the tails of the sigmoid --------------------------------------------------------------------------
def _tail_inputs(dev, B, T, D, t, seed):
    """Gates from -104 to -80 and from 80 to 104 in steps of 1/16, far ones, infinities, and a few moderate ones in between.
    Only one of a and 1 - a is there in 32 bits (the other one's exponential may be flushed below 2^-126): with |x|, |h| <= 1/2
    and |e| <= 1 what is flushed is at most 2^-126 of any result, and `store` grants 2^-125."""
    g = _gen(dev, seed)
    near = torch.arange(80, 104, 1 / 16)
    values = torch.cat([-near, -near, near, torch.tensor([-1e4, 1e4, -110.0, 110.0, float("-inf"), float("inf")] * 16)]).to(dev)
    gate = values[torch.randint(0, len(values), (B, T, D), generator=g, device=dev)]
    some = torch.rand(B, T, D, generator=g, device=dev) < 0.2
    gate = torch.where(some, 3 * torch.randn(B, T, D, generator=g, device=dev), gate).to(t)
    x, dy = ((torch.rand(B, T, D, generator=g, device=dev) - 0.5).to(t) for _ in range(2))
    h0, dl = (torch.rand(B, D, generator=g, device=dev) - 0.5 for _ in range(2))
    return gate, x, (dy / 32).to(t), h0, dl / 32


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,T,D", [(64, 1, 40), (3, 40, 33), (2, 300, 64), (3, 300, 34), (2, 530, 72), (40, 513, 256), (1, 4096, 64), (1, 3001, 33)])
def test_gates_in_the_tails(dev, B, T, D, kind):
    """single steps, staged pieces, tiles, and both shared by the blocks of a cluster"""
    gate, x, dy, h0, dl = _tail_inputs(dev, B, T, D, TYPES[kind], 51)
    sens = lm.gated_recurrence_backward(gate, x, h0, dy, dl)[3]
    assert sens.abs().max() <= 1
    h, _, _ = _check_rec(ops, gate, x, dy, h0, dl)
    reset = gate <= -104
    assert torch.equal(h[reset], x[reset])


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("gate", [-87.5, -88.0, -88.5, -87.0, -89.0])
def test_a_gate_that_leaves_nothing_of_the_state(dev, gate, kind):
    for T in (1, 20, 600):
        x = torch.randn(2, T, 64, generator=_gen(dev, 52), device=dev).to(TYPES[kind])
        g = torch.full_like(x, gate)
        h, last, states = ops.gated_recurrence(g, x, None, True)
        # 1 - a is 1 up to the roundings of e, of the sum, of the reciprocal and of the product: 8 half steps
        assert ((h.double() - x.double()).abs() <= lm.store(8 * lm.U * x.double().abs(), x.double(), x.dtype)).all()
        _, dx, _ = ops.gated_recurrence_backward(g, x, states, x)
        assert ((dx.double() - x.double()).abs() <= lm.store(8 * lm.U * x.double().abs(), x.double(), x.dtype)).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("T", [1, 20, 600])
def test_a_gate_that_is_no_number(dev, T, kind):
    g = _gen(dev, 53)
    gate, x, dy = (torch.randn(2, T, 64, generator=g, device=dev).to(TYPES[kind]) for _ in range(3))
    at = T // 2
    gate[1, at, 5] = float("nan")
    h, last, states = ops.gated_recurrence(gate, x, None, True)
    dg, dx, dh0 = ops.gated_recurrence_backward(gate, x, states, dy)
    for got in (h[1, at:, 5], last[1, 5], dg[1, :at + 1, 5], dx[1, :at + 1, 5], dh0[1, 5]):
        assert got.isnan().all()
    assert h.isnan().sum() == T - at and dx.isnan().sum() == at + 1


# ---- rows that no kernel takes ----------------------------------------------------------------------------------
def test_rows_whose_length_passes_32_bits_are_refused(dev, api):
    """not taken for rows of the length's lower 32 bits"""
    x = torch.zeros(1, (1 << 32) + 8, dtype=torch.float16, device=dev)
    ids, one = torch.zeros(1, dtype=torch.int64, device=dev), torch.ones(1, device=dev)
    for call in (lambda: api.layer_norm(x), lambda: api.layer_norm_backward(x, x, one, one), lambda: api.embedding(x, ids),
                 lambda: api.embedding_backward(x, ids, 1), lambda: api.gated_recurrence(x[None], x[None]),
                 lambda: api.gated_recurrence_backward(x[None], x[None], x[None].view(torch.float32), x[None])):
        with pytest.raises((ValueError, RuntimeError), match="too long rows"):
            call()


# ---- infinite gradients -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,D", [(300, 40), (300, 304), (500, 1000), (300, 2050), (400, 1001), (300, 515), (200, 8190), (130, 16400), (20, 1000)])
@pytest.mark.parametrize("weighted", [True, False])
def test_layer_norm_gradient_of_rows_with_infinite_elements(dev, rows, D, kind, weighted):
    """What the definition gives for a row whose gradient is infinite in its last or first element: an infinite element
    where all terms agree in sign, no number elsewhere; rows without one are not touched."""
    g = _gen(dev, 54)
    x, dy = (torch.randn(rows, D, generator=g, device=dev).to(TYPES[kind]) for _ in range(2))
    w = 1 + torch.rand(D, generator=g, device=dev) if weighted else None
    _, mean, invstd = ops.layer_norm(x, w)
    ref = ops.layer_norm_backward(x, dy, mean, invstd, w)
    at = torch.arange(rows, device=dev)
    bad = dy.clone()
    bad[at % 5 == 1, -1], bad[at % 5 == 3, 0] = float("inf"), float("-inf")
    dx, dw, db = ops.layer_norm_backward(x, bad, mean, invstd, w)
    exact = lm.layer_norm_backward(x, bad, mean, invstd, w)
    hit = (at % 5 == 1) | (at % 5 == 3)
    assert torch.equal(dx[~hit], ref[0][~hit]) and exact[0][hit].isinf().any() and exact[2][-1] == float("inf")
    for got, want in ((dx[hit], exact[0][hit]), (dw[[0, -1]], exact[1][[0, -1]]), (db[[0, -1]], exact[2][[0, -1]])):
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got[want.isinf()].double(), want[want.isinf()])
    assert torch.equal(dw[1:-1], ref[1][1:-1]) and torch.equal(db[1:-1], ref[2][1:-1])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,D", [(300, 40), (300, 304), (500, 1000), (400, 1001), (300, 515), (200, 8190), (130, 16400), (20, 1000)])
def test_layer_norm_gradient_of_large_constant_rows(dev, rows, D, kind):
    """Rows of one value: x - mean is zero, whatever mean times invstd is.  2^123 / sqrt(1e-5) is beyond 32 bits; the sums of D such
    values are not (a power of two, so that they are exact)."""
    dy = torch.randn(rows, D, generator=_gen(dev, 55), device=dev).to(TYPES[kind])
    big = torch.full_like(dy, 2.0 ** 123)
    mean, invstd = torch.full((rows,), 2.0 ** 123, device=dev), torch.full((rows,), 1e-5 ** -0.5, device=dev)
    small = torch.zeros_like(dy), torch.zeros_like(mean)
    for got, want in zip(ops.layer_norm_backward(big, dy, mean, invstd), ops.layer_norm_backward(small[0], dy, small[1], invstd)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("D", [301, 1000, 2050])
def test_layer_norm_gradient_with_infinite_elements_of_tensors_that_begin_anywhere(dev, D, kind):
    """single elements: x and grad_out begin unequally far behind an aligned address"""
    g = _gen(dev, 56)
    flat = torch.randn(2, 400 * D + 8, generator=g, device=dev).to(TYPES[kind])
    x, dy = flat[0, 1:400 * D + 1].view(400, D), flat[1, 2:400 * D + 2].view(400, D)
    _, mean, invstd = ops.layer_norm(x)
    dy[::3, -1] = float("inf")
    dx = ops.layer_norm_backward(x, dy, mean, invstd)[0]
    exact = lm.layer_norm_backward(x, dy, mean, invstd, None)[0]
    assert torch.equal(dx.isnan(), exact.isnan()) and torch.equal(dx[exact.isinf()].double(), exact[exact.isinf()])
    assert exact.isinf().any() and dx[1::3].isfinite().all()


# ---- sums that are exact in 32 bits -----------------------------------------------------------------------------
@pytest.mark.parametrize("n,V,D,how,kind", [
    (200, 3, 40, "even", "bf16"), (1000, 1, 8, "one", "f32"), (1000, 1, 33, "one", "f16"), (8192, 5, 64, "one", "bf16"), (8192, 40, 7, "text", "f32"),
    (17000, 3, 24, "one", "f32"), (17600, 3, 25, "one", "bf16"), (20000, 2, 64, "even", "f16"), (32769, 2, 64, "one", "bf16"),
    (40000, 4, 24, "one", "f32"), (40000, 3, 9, "even", "f32"), (70000, 3, 128, "one", "f16"), (70000, 1000, 64, "text", "f32"),
    (300000, 2, 8, "even", "f32"), (300000, 7, 8, "text", "bf16"), (300000, 50000, 16, "text", "f16"), (1 << 20, 3, 4, "one", "f32")])
def test_embedding_gradient_without_a_lost_or_doubled_token(dev, n, V, D, how, kind):
    """Whole numbers up to 8, no sum beyond 2^24: every order of additions gives the same bits, so nothing may be off.
    Runs of more than 33 chunks and of more than 545, where the join looks for their ends in steps of 512."""
    ids = _ids(dev, n, V, how, 57)
    ids[7::1000], ids[11::1300] = -1, V
    dy = torch.randint(-8, 9, (n, D), generator=_gen(dev, 58), device=dev).to(TYPES[kind])
    assert torch.equal(ops.embedding_backward(dy, ids, V, 0.5), lm.embedding_backward(dy, ids, V, 0.5).to(TYPES[kind]))
    assert torch.equal(ops.embedding_backward(dy, ids, V, 2.0, V // 2), lm.embedding_backward(dy, ids, V, 2.0, V // 2).to(TYPES[kind]))
