"""The language-model operators against their 64-bit definitions, inside the bounds that 32-bit arithmetic gives."""
import pytest
import torch

from hfuse_b200 import _lib, ops
from oracle import lm

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def within(got, exact, bound, dtype=None):
    """got is of type dtype and no further from exact than the bound and one rounding to that type allow"""
    dtype = dtype or got.dtype
    assert got.dtype == dtype and got.shape == exact.shape
    off, may = (got.double() - exact).abs(), lm.store(bound, exact, dtype)
    assert (off <= may).all(), f"{(off / may).max().item():.3g} times the bound"


@pytest.fixture(params=["harness", "extension"])
def api(request):
    """Both Python entry points with one signature."""
    if request.param == "harness":
        return ops
    from hfuse_b200 import torch_ops

    class Extension:
        layer_norm = staticmethod(lambda x, w=None, b=None, eps=1e-5: torch_ops.ops.layer_norm(x, w, b, eps))
        layer_norm_backward = staticmethod(lambda x, dy, m, r, w=None: torch_ops.ops.layer_norm_backward(x, dy, m, r, w))
        embedding = staticmethod(lambda t, i, s=1.0: torch_ops.ops.embedding(t, i, s))
        embedding_backward = staticmethod(lambda dy, i, rows, s=1.0, pad=-1: torch_ops.ops.embedding_backward(dy, i, rows, s, pad))
        gated_recurrence = staticmethod(lambda g, x, h=None, save=False: torch_ops.ops.gated_recurrence(g, x, h, save))
        gated_recurrence_backward = staticmethod(lambda g, x, s, dy, dl=None: torch_ops.ops.gated_recurrence_backward(g, x, s, dy, dl))

    return Extension


# ---- layer norm -------------------------------------------------------------------------------------------------
NORM_SHAPES = [(1, 1), (1, 4096), (3, 7), (5, 32), (700, 64), (37, 129), (2, 1001), (333, 1000), (64, 2048), (300, 512), (9, 8192),
               (5, 8190), (3, 16384), (3, 20000), (2, 70001), (2500, 96), (5000, 24), (1200, 256), (450, 1024), (301, 4095),
               (600, 4096), (601, 1001), (700, 2050), (300, 8192), (257, 8191), (130, 16384), (100, 24576)]


def _norm_inputs(dev, rows, D, t, wt, seed, offset=0.3):
    g = _gen(dev, seed)
    x = (offset + torch.randn(rows, D, generator=g, device=dev) * (0.5 + torch.rand(rows, 1, generator=g, device=dev))).to(t)
    w = (1 + 0.3 * torch.randn(D, generator=g, device=dev)).to(wt)
    b = (0.3 * torch.randn(D, generator=g, device=dev)).to(wt)
    return x, w, b, torch.randn(rows, D, generator=g, device=dev).to(t)


def _check_norm(api, x, w, b, dy, eps=1e-5):
    y, mean, invstd = api.layer_norm(x, w, b, eps)
    wt = w.dtype if w is not None else b.dtype if b is not None else x.dtype
    for got, exact, bound, t in zip((y, mean, invstd), lm.layer_norm(x, w, b, eps), lm.layer_norm_bound(x, w, b, eps),
                                    (x.dtype, torch.float32, torch.float32)):
        within(got, exact, bound, t)
    grads = api.layer_norm_backward(x, dy, mean, invstd, w)
    wt = w.dtype if w is not None else x.dtype
    for got, exact, bound, t in zip(grads, lm.layer_norm_backward(x, dy, mean, invstd, w),
                                    lm.layer_norm_backward_bound(x, dy, mean, invstd, w), (x.dtype, wt, wt)):
        within(got, exact, bound, t)
    return (y, mean, invstd) + tuple(grads)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,D", NORM_SHAPES)
def test_layer_norm(dev, rows, D, kind):
    x, w, b, dy = _norm_inputs(dev, rows, D, TYPES[kind], TYPES[kind], 11)
    _check_norm(ops, x, w, b, dy)


@pytest.mark.parametrize("rows,D,kind", [(40, 768, "bf16"), (7, 1001, "f16"), (1500, 64, "bf16"), (3, 20000, "f16")])
def test_layer_norm_under_float_weights(dev, api, rows, D, kind):
    x, w, b, dy = _norm_inputs(dev, rows, D, TYPES[kind], torch.float32, 12)
    _check_norm(api, x, w, b, dy)


@pytest.mark.parametrize("D", [64, 33, 2048])
def test_layer_norm_without_weight_or_bias(dev, api, D):
    x, w, b, dy = _norm_inputs(dev, 50, D, torch.bfloat16, torch.bfloat16, 13)
    _check_norm(api, x, None, None, dy)
    _check_norm(api, x, None, b, dy)
    _check_norm(api, x, w, None, dy)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("at,D,wide", [(8, 64, 192), (3, 64, 200), (64, 1024, 2048), (1, 1024, 1500), (0, 129, 131)])
def test_layer_norm_of_a_slice_of_wider_rows(dev, api, at, D, wide, kind):
    big, _, _, dbig = _norm_inputs(dev, 6 * 35, wide, TYPES[kind], TYPES[kind], 14)
    _, w, b, _ = _norm_inputs(dev, 1, D, TYPES[kind], TYPES[kind], 15)
    x, dy = big.view(6, 35, wide)[..., at:at + D], dbig.view(6, 35, wide)[..., at:at + D]
    got = _check_norm(api, x, w, b, dy)
    assert got[0].is_contiguous() and got[0].shape == x.shape
    with pytest.raises((ValueError, RuntimeError), match="evenly spaced"):
        api.layer_norm(big.view(6, 35, wide)[:, :20, at:at + D], w, b)
    with pytest.raises((ValueError, RuntimeError), match="stride 1"):
        api.layer_norm(big.t(), None, None)


def test_layer_norm_far_from_zero_and_of_constant_rows(dev):
    x, w, b, dy = _norm_inputs(dev, 64, 1024, torch.float32, torch.float32, 16, offset=1000.0)
    _check_norm(ops, x, w, b, dy)
    y, mean, invstd = ops.layer_norm(torch.full((4, 512), 3.0, device=dev), None, None, 1e-5)
    assert (y == 0).all() and (mean == 3).all()
    torch.testing.assert_close(invstd, torch.full((4,), 1e-5 ** -0.5, device=dev), rtol=4 * lm.U, atol=0)


def test_layer_norm_keeps_a_bad_row_to_itself(dev):
    x, w, b, dy = _norm_inputs(dev, 90, 256, torch.bfloat16, torch.bfloat16, 17)
    good = ops.layer_norm(x, w, b)
    bad = x.clone()
    bad[7, 3], bad[50, 0], bad[89, 255] = float("nan"), float("inf"), float("-inf")
    y, mean, invstd = ops.layer_norm(bad, w, b)
    rows = torch.tensor([7, 50, 89], device=dev)
    keep = torch.ones(90, dtype=torch.bool, device=dev)
    keep[rows] = False
    assert y[rows].isnan().all() and torch.equal(y[keep], good[0][keep]) and torch.equal(mean[keep], good[1][keep])
    dx, dw, db = ops.layer_norm_backward(bad, dy, mean, invstd, w)
    ref = ops.layer_norm_backward(x, dy, good[1], good[2], w)
    assert torch.equal(dx[keep], ref[0][keep]) and dx[rows].isnan().all() and torch.equal(db, ref[2])


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("rows", [1, 5, 7, 300, 1201])
@pytest.mark.parametrize("D,wide", [(129, 193), (1001, 1009), (2047, 4095)])
def test_layer_norm_of_a_slice_with_rows_of_equal_offset(dev, rows, D, wide, kind):
    t = TYPES[kind]
    x, w, b, dy = _norm_inputs(dev, rows, D, t, torch.float32, 37)
    room = torch.full((rows, wide), float("nan"), dtype=t, device=dev)
    grads = room.clone()
    room[:, :D], grads[:, :D] = x, dy
    got, ref = _check_norm(ops, room[:, :D], w, b, grads[:, :D]), _check_norm(ops, x, w, b, dy)
    for g, r in zip(got[:4], ref[:4]):
        assert torch.equal(g, r)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("D", [1001, 250, 333])
def test_layer_norm_keeps_bad_rows_to_themselves_where_rows_share_accesses(dev, D, kind):
    x, w, b, dy = _norm_inputs(dev, 1500, D, TYPES[kind], torch.float32, 29)
    ref = _check_norm(ops, x, w, b, dy)
    rows = torch.arange(3, 1500, 7, device=dev)
    bx, bd, keep = x.clone(), dy.clone(), torch.ones(1500, dtype=torch.bool, device=dev)
    keep[rows] = False
    bx[rows], bd[rows] = float("inf"), float("nan")
    y, mean, invstd = ops.layer_norm(bx, w, b)
    assert torch.equal(y[keep], ref[0][keep]) and torch.equal(mean[keep], ref[1][keep]) and y[rows].isnan().all()
    dx, _, _ = ops.layer_norm_backward(bx, bd, mean, invstd, w)
    assert torch.equal(dx[keep], ref[3][keep]) and dx[rows].isnan().all()


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("rows,D,at", [(300, 1001, (1, 1)), (300, 1001, (1, 2)), (1100, 512, (3, 3)), (400, 2046, (0, 0)), (5000, 515, (2, 2))])
def test_layer_norm_of_tensors_that_begin_anywhere(dev, rows, D, at, kind):
    """rows that begin equally or unequally far behind an aligned address, nothing behind them touched"""
    def place(t, k):
        flat = torch.full((t.numel() + 8,), 7.0, dtype=t.dtype, device=dev)
        flat[k:k + t.numel()] = t.flatten()
        return flat, flat[k:k + t.numel()].view(t.shape)

    x, w, b, dy = _norm_inputs(dev, rows, D, TYPES[kind], torch.float32, 31)
    (fx, px), (fd, pd) = place(x, at[0]), place(dy, at[1])
    _check_norm(ops, px, w, b, pd)
    # outputs placed by the caller too
    m, r = lm.layer_norm(x, w, b, 1e-5)[1:]
    m, r = m.float(), r.float()
    (fg, pg), dw, db = place(torch.empty_like(x), at[0]), torch.empty(D, device=dev), torch.empty(D, device=dev)
    L = _lib.lib()
    ws = torch.empty(L.hfuse_layernorm_backward_workspace_bytes(rows, D), dtype=torch.uint8, device=dev)
    t = ops._LM_TYPES[x.dtype]
    _lib.check(L.hfuse_layernorm_backward(px.data_ptr(), D, pd.data_ptr(), D, rows, D, t, m.data_ptr(), r.data_ptr(), w.data_ptr(), 0,
                                          pg.data_ptr(), dw.data_ptr(), db.data_ptr(), ws.data_ptr(), ws.numel(),
                                          torch.cuda.current_stream().cuda_stream), "hfuse_layernorm_backward")
    for got, exact, bound in zip((pg, dw, db), lm.layer_norm_backward(x, dy, m, r, w), lm.layer_norm_backward_bound(x, dy, m, r, w)):
        within(got, exact, bound)
    assert (fg[:at[0]] == 7).all() and (fg[at[0] + x.numel():] == 7).all()


def test_layer_norm_of_no_rows(dev, api):
    x, w = torch.empty(0, 16, device=dev), torch.ones(16, device=dev)
    y, mean, invstd = api.layer_norm(x, w, None)
    assert y.shape == (0, 16) and mean.shape == (0,)
    dx, dw, db = api.layer_norm_backward(x, x, mean, invstd, w)
    assert dx.shape == (0, 16) and (dw == 0).all() and (db == 0).all()


@pytest.mark.parametrize("shape", [(5, 0, 16), (0, 5, 16), (2, 0, 3, 16)])
def test_layer_norm_of_an_empty_batch(dev, api, shape):
    x, w = torch.empty(shape, device=dev), torch.ones(16, device=dev)
    y, mean, invstd = api.layer_norm(x, w, w)
    assert y.shape == x.shape and mean.shape == invstd.shape == x.shape[:-1]
    dx, dw, db = api.layer_norm_backward(x, x, mean, invstd, w)
    assert dx.shape == x.shape and (dw == 0).all() and (db == 0).all()


def test_layer_norm_shapes_and_refusals(dev, api):
    x = torch.randn(2, 3, 5, 16, device=dev)
    y, mean, _ = api.layer_norm(x)
    assert y.shape == x.shape and mean.shape == (2, 3, 5)
    v, vm, _ = api.layer_norm(x[0, 0, 0])
    assert v.shape == (16,) and vm.shape == () and torch.equal(v, y[0, 0, 0])
    w = torch.ones(16, device=dev)
    for bad in (lambda: api.layer_norm(x, w[:15]), lambda: api.layer_norm(x, w.double()), lambda: api.layer_norm(x.int()),
                lambda: api.layer_norm(x.bfloat16(), w.half()), lambda: api.layer_norm(x, w, None, -1.0),
                lambda: api.layer_norm(x, w.cpu()), lambda: api.layer_norm(x[..., :1].expand(2, 3, 5, 16)),
                lambda: api.layer_norm(x[:1, :1, :1].expand(2, 3, 5, 16)),
                lambda: api.layer_norm_backward(x, x[:1], mean, mean, w), lambda: api.layer_norm_backward(x, x, mean[0], mean, w),
                lambda: api.layer_norm_backward(x, x.half(), mean, mean, w),
                lambda: api.layer_norm_backward(x, x, mean.half(), mean, w)):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            bad()


# ---- embedding --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape,V,D", [((1,), 1, 1), ((3, 5), 7, 8), ((1000,), 300, 33), ((64,), 32000, 1024), ((7, 129), 1001, 250),
                                       ((5000,), 50, 64), ((2,), 5, 20000)])
def test_embedding(dev, api, shape, V, D, kind):
    g = _gen(dev, 21)
    table = torch.randn(V, D, generator=g, device=dev).to(TYPES[kind])
    ids = torch.randint(0, V, shape, generator=g, device=dev)
    want = (table[ids].float() * 1.7).to(table.dtype)              # one product, one rounding: the same bits
    scale = float(torch.tensor(1.7, dtype=torch.float32))
    assert torch.equal(api.embedding(table, ids, scale), want)
    assert torch.equal(api.embedding(table, ids.int(), scale), want)
    within(want, lm.embedding(table, ids, scale), lm.U * lm.embedding(table, ids, scale).abs())


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("D", [16, 31, 32, 33, 35, 64, 250, 1001, 2046, 4097])
@pytest.mark.parametrize("at", [(0, 0), (1, 0), (3, 3), (2, 5), (7, 4)])
def test_embedding_of_tables_and_outputs_that_begin_anywhere(dev, D, at, kind):
    V, t = 9, TYPES[kind]
    flat = torch.randn(V * D + 16, generator=_gen(dev, 41), device=dev).to(t)
    flat[:at[0]], flat[at[0] + V * D:] = float("nan"), float("nan")
    table = flat[at[0]:at[0] + V * D].view(V, D)
    ids = torch.tensor([0, V - 1, 4, 4, -1, V, 3, 0, V - 1, 7, 1], dtype=torch.int32, device=dev)
    room = torch.full((len(ids) * D + 16,), 7.0, dtype=t, device=dev)
    out = room[at[1]:at[1] + len(ids) * D].view(len(ids), D)
    _lib.check(_lib.lib().hfuse_embedding(table.data_ptr(), V, D, ops._LM_TYPES[t], ids.data_ptr(), len(ids), 4, 1.5, out.data_ptr(),
                                          torch.cuda.current_stream().cuda_stream), "hfuse_embedding")
    exact = torch.where(((ids >= 0) & (ids < V))[:, None], table[ids.clamp(0, V - 1).long()].double() * 1.5, 0.0)
    assert torch.equal(out, exact.to(t))              # a product with 1.5 of a 16-bit value is exact in 32 bits, of a float one rounding
    assert (room[:at[1]] == 7).all() and (room[at[1] + len(ids) * D:] == 7).all()


def test_embedding_ids_outside_the_table(dev, api):
    table = torch.randn(10, 24, device=dev)
    ids = torch.tensor([0, -1, 9, 10, 1 << 40, -(1 << 40), 5], device=dev)
    out = api.embedding(table, ids, 2.0)
    assert torch.equal(out, lm.embedding(table, ids, 2.0).float())
    assert api.embedding(table, ids[:0], 2.0).shape == (0, 24)
    dy = torch.randn(7, 24, device=dev)
    grad = api.embedding_backward(dy, ids, 10, 2.0)
    assert torch.equal(grad, lm.embedding_backward(dy, ids, 10, 2.0).float())
    assert (api.embedding_backward(dy[:0], ids[:0], 10, 2.0) == 0).all()


def _ids(dev, n, V, how, seed):
    g = _gen(dev, seed)
    if how == "one":
        return torch.full((n,), V // 2, device=dev, dtype=torch.int64)
    if how == "rising":
        return torch.arange(n, device=dev) % V
    if how == "text":
        r = torch.exp(torch.rand(n, generator=g, device=dev, dtype=torch.float64) * torch.log(torch.tensor(V + 1.0))) - 1
        return torch.randperm(V, generator=g, device=dev)[r.long().clamp(0, V - 1)]
    return torch.randint(0, V, (n,), generator=g, device=dev)


@pytest.mark.parametrize("n,V,D,how,kind", [
    (1, 1, 1, "one", "f32"), (2, 511, 8, "even", "bf16"), (31, 512, 16, "even", "f16"), (32, 513, 33, "one", "bf16"),
    (33, 3, 64, "one", "f32"), (64, 2, 8, "rising", "f32"), (65, 64, 8, "rising", "f16"), (2047, 1000, 40, "text", "f32"),
    (2048, 262143, 8, "even", "bf16"), (2049, 262144, 8, "even", "f32"), (4100, 50257, 1001, "text", "f16"),
    (5000, 100, 128, "text", "bf16"), (255, 60, 65, "text", "bf16"), (256, 9, 40, "one", "f16"), (257, 60, 65, "text", "f32"),
    (8192, 4000, 48, "text", "bf16"), (8193, 4000, 50, "text", "f16"), (200, 600000, 8, "even", "bf16"), (8000, 300000, 8, "even", "f16"),
 (70000, 30000, 64, "text", "bf16"), (40000, 4, 24, "one", "f32"), (300000, 1000, 8, "text", "f32"),
    (300000, 7, 8, "even", "bf16"), (777, 1 << 20, 9, "even", "f32"), (16384, 32000, 512, "text", "f16"), (9000, 9000, 2048, "rising", "bf16")])
def test_embedding_backward(dev, n, V, D, how, kind):
    ids = _ids(dev, n, V, how, 22)
    dy = torch.randn(n, D, generator=_gen(dev, 23), device=dev).to(TYPES[kind])
    got = ops.embedding_backward(dy, ids, V, 0.5)
    within(got, lm.embedding_backward(dy, ids, V, 0.5), lm.embedding_backward_bound(dy, ids, V, 0.5), TYPES[kind])
    assert torch.equal(got, ops.embedding_backward(dy, ids.int(), V, 0.5))           # the same bits every time


@pytest.mark.parametrize("pad", [0, 17, 99])
def test_embedding_backward_padding_and_unused_ids(dev, api, pad):
    ids = _ids(dev, 6000, 100, "text", 24)
    ids[::3] = pad
    ids[1::50], ids[2::70] = -5, 100
    dy = torch.randn(6000, 72, generator=_gen(dev, 25), device=dev).bfloat16()
    got = api.embedding_backward(dy.view(60, 100, 72), ids.view(60, 100), 100, 3.0, pad)
    within(got, lm.embedding_backward(dy, ids, 100, 3.0, pad), lm.embedding_backward_bound(dy, ids, 100, 3.0, pad))
    assert (got[pad] == 0).all()


def test_embedding_backward_of_padding_alone(dev, api):
    ids = torch.full((3000,), 4, device=dev)
    assert (api.embedding_backward(torch.randn(3000, 16, device=dev), ids, 9, 1.0, 4) == 0).all()


def test_embedding_refusals(dev, api):
    table, ids = torch.randn(10, 24, device=dev), torch.zeros(4, dtype=torch.int64, device=dev)
    dy = torch.randn(4, 24, device=dev)
    for bad in (lambda: api.embedding(table.t(), ids), lambda: api.embedding(table[0], ids), lambda: api.embedding(table, ids.short()),
                lambda: api.embedding(table, ids.cpu()), lambda: api.embedding(table, torch.zeros(8, dtype=torch.int64, device=dev)[::2]),
                lambda: api.embedding(table[:0], ids), lambda: api.embedding(table.double(), ids),
                lambda: api.embedding_backward(dy, ids[:3], 10), lambda: api.embedding_backward(dy, ids, 0),
                lambda: api.embedding_backward(dy[:, ::2], ids, 10), lambda: api.embedding_backward(dy.double(), ids, 10)):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            bad()


# ---- gated recurrence -------------------------------------------------------------------------------------------
def _rec_inputs(dev, B, T, D, t, seed):
    g = _gen(dev, seed)
    gate = (2 + 2.5 * torch.randn(B, T, D, generator=g, device=dev)).to(t)
    x, dy = (torch.randn(B, T, D, generator=g, device=dev).to(t) for _ in range(2))
    h0, dl = (torch.randn(B, D, generator=g, device=dev) for _ in range(2))
    return gate, x, dy, h0, dl


def _check_rec(api, gate, x, dy, h0, dl):
    h, last, states = api.gated_recurrence(gate, x, h0, True)
    eh, before, elast = lm.gated_recurrence(gate, x, h0)
    bh, bbefore, blast = lm.gated_recurrence_bound(gate, x, h0)
    within(h, eh, bh, x.dtype)
    within(last, elast, blast, torch.float32)
    step = _lib.HFUSE_RECURRENCE_CHUNK
    within(states, before[:, ::step], bbefore[:, ::step], torch.float32)
    plain = api.gated_recurrence(gate, x, h0)
    assert torch.equal(plain[0], h) and torch.equal(plain[1], last) and plain[2].numel() == 0
    grads = api.gated_recurrence_backward(gate, x, states, dy, dl)
    for got, exact, bound, t in zip(grads, lm.gated_recurrence_backward(gate, x, h0, dy, dl),
                                    lm.gated_recurrence_backward_bound(gate, x, h0, dy, dl), (x.dtype, x.dtype, torch.float32)):
        within(got, exact, bound, t)
    return h, last, states


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,T,D", [(1, 1, 1), (2, 1, 64), (64, 1, 257), (1, 2, 3), (3, 15, 32), (2, 16, 33), (5, 17, 34), (3, 255, 33),
                                   (2, 256, 64), (2, 257, 40), (1, 513, 130), (300, 5, 8), (4, 700, 96), (1, 3001, 8), (2, 1500, 66), (3, 2049, 64), (1, 4096, 200), (40, 513, 256)])
def test_gated_recurrence(dev, B, T, D, kind):
    gate, x, dy, h0, dl = _rec_inputs(dev, B, T, D, TYPES[kind], 31)
    _check_rec(ops, gate, x, dy, h0, dl)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_gated_recurrence_from_nothing(dev, api, kind):
    gate, x, dy, _, _ = _rec_inputs(dev, 2, 300, 48, TYPES[kind], 32)
    _check_rec(api, gate, x, dy, None, None)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("D,at", [(64, 0), (64, 3), (33, 0), (250, 2)])
def test_gated_recurrence_of_halves_of_one_buffer(dev, api, D, at, kind):
    g = _gen(dev, 33)
    both = torch.randn(2, 333, 2 * D + 6, generator=g, device=dev).to(TYPES[kind])
    gate, x = both[..., at:at + D], both[..., at + D:at + 2 * D]
    dy = torch.randn(333, 2, D, generator=g, device=dev).to(TYPES[kind]).transpose(0, 1)
    h0, dl = (torch.randn(2, D, generator=g, device=dev) for _ in range(2))
    _check_rec(api, gate, x, dy, h0, dl)
    # a gate that all sequences share
    _check_rec(api, gate[:1].expand(2, 333, D), x, dy, h0, dl)


def test_gated_recurrence_in_pieces_and_single_steps(dev, api):
    gate, x, _, h0, _ = _rec_inputs(dev, 3, 600, 80, torch.bfloat16, 34)
    whole, last, _ = api.gated_recurrence(gate, x, h0)
    bound = lm.gated_recurrence_bound(gate, x, h0)
    exact = lm.gated_recurrence(gate, x, h0)
    h, out = h0, []
    for a, b in ((0, 1), (1, 2), (2, 300), (300, 557), (557, 600)):
        y, h, _ = api.gated_recurrence(gate[:, a:b], x[:, a:b], h)
        out.append(y)
    within(torch.cat(out, 1), exact[0], bound[0])
    within(h, exact[2], bound[2])


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_gates_of_infinity(dev, api, kind):
    gate, x, dy, h0, dl = _rec_inputs(dev, 2, 530, 36, TYPES[kind], 35)
    gate[:, 100], gate[:, 256], gate[0, 511] = float("-inf"), float("-inf"), float("-inf")
    gate[:, 101:140], gate[1, 300:400] = float("inf"), float("inf")
    h, _, _ = _check_rec(api, gate, x, dy, h0, dl)
    assert torch.equal(h[:, 100], x[:, 100]) and torch.equal(h[:, 139], x[:, 100]) and torch.equal(h[:, 256], x[:, 256])


def test_gated_recurrence_keeps_a_bad_channel_to_itself(dev):
    gate, x, dy, h0, dl = _rec_inputs(dev, 2, 400, 70, torch.float32, 36)
    h, last, states = ops.gated_recurrence(gate, x, h0, True)
    ref = ops.gated_recurrence_backward(gate, x, states, dy, dl)
    bg, bx = gate.clone(), x.clone()
    bg[0, 50, 3], bx[1, 399, 69] = float("nan"), float("inf")
    h2, last2, states2 = ops.gated_recurrence(bg, bx, h0, True)
    keep = torch.ones(2, 70, dtype=torch.bool, device=dev)
    keep[0, 3] = keep[1, 69] = False
    pick = keep[:, None, :].expand(2, 400, 70)
    assert torch.equal(h2[pick], h[pick]) and torch.equal(last2[keep], last[keep])
    assert torch.equal(h2[0, :50, 3], h[0, :50, 3]) and h2[0, 50:, 3].isnan().all()
    got = ops.gated_recurrence_backward(bg, bx, states2, dy, dl)
    assert torch.equal(got[0][pick], ref[0][pick]) and torch.equal(got[1][pick], ref[1][pick])


def test_gated_recurrence_refusals(dev, api):
    g = torch.randn(2, 5, 8, device=dev)
    st = torch.zeros(2, 1, 8, device=dev)
    for bad in (lambda: api.gated_recurrence(g, g[:, :4]), lambda: api.gated_recurrence(g, g.half()), lambda: api.gated_recurrence(g[0], g[0]),
                lambda: api.gated_recurrence(g, g, torch.zeros(2, 7, device=dev)), lambda: api.gated_recurrence(g, g, st[:, 0].half()),
                lambda: api.gated_recurrence(g[:, :0], g[:, :0]), lambda: api.gated_recurrence(g.transpose(1, 2), g.transpose(1, 2)),
                lambda: api.gated_recurrence(g, g.cpu()), lambda: api.gated_recurrence_backward(g, g, st[:, :, :7], g),
                lambda: api.gated_recurrence_backward(g, g, st, g[:1]), lambda: api.gated_recurrence_backward(g, g, st, g, st)):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            bad()


# ---- more than 2^31 elements ------------------------------------------------------------------------------------
def test_layer_norm_beyond_32_bits(dev):
    rows, D, last = 1_100_000, 2048, 96
    x, dy = torch.zeros(rows, D, dtype=torch.float16, device=dev), torch.zeros(rows, D, dtype=torch.float16, device=dev)
    xs, w, b, dys = _norm_inputs(dev, last, D, torch.float16, torch.float16, 18)
    x[-last:], dy[-last:] = xs, dys
    y, mean, invstd = ops.layer_norm(x, w, b)
    for got, exact, bound in zip((y[-last:], mean[-last:], invstd[-last:]), lm.layer_norm(xs, w, b, 1e-5), lm.layer_norm_bound(xs, w, b, 1e-5)):
        within(got, exact, bound)
    del y
    dx, dw, db = ops.layer_norm_backward(x, dy, mean, invstd, w)
    m, r = mean[-last:], invstd[-last:]
    # all other rows add zeros
    for got, exact, bound in zip((dx[-last:], dw, db), lm.layer_norm_backward(xs, dys, m, r, w), lm.layer_norm_backward_bound(xs, dys, m, r, w)):
        within(got, exact, bound)
    assert (dx[:64] == 0).all()


def test_embedding_beyond_32_bits(dev):
    V, D = 70_000, 32_768
    ids = torch.tensor([V - 1, 3, V - 2, V - 1, 66_000] * 60, device=dev)
    table = torch.zeros(V, D, dtype=torch.float16, device=dev)
    rows = torch.unique(ids)
    table[rows] = torch.randn(len(rows), D, generator=_gen(dev, 26), device=dev).half()
    assert torch.equal(ops.embedding(table, ids[:7], 2.0), (table[ids[:7]].float() * 2).half())
    del table
    dy = torch.randn(300, D, generator=_gen(dev, 27), device=dev).half()
    grad = ops.embedding_backward(dy, ids, V)
    small = torch.searchsorted(rows, ids)
    within(grad[rows], lm.embedding_backward(dy, small, len(rows), 1.0), lm.embedding_backward_bound(dy, small, len(rows), 1.0))
    grad[rows] = 0
    assert not grad.any()


def test_gated_recurrence_beyond_32_bits(dev):
    B, T, D, pick = 2, 4100, 270_336, slice(270_336 - 64, 270_336)
    g = _gen(dev, 37)
    gate, x = (torch.randn(B, T, D, generator=g, device=dev, dtype=torch.float16) for _ in range(2))
    h, last, states = ops.gated_recurrence(gate, x, None, True)
    gs, xs = gate[..., pick].contiguous(), x[..., pick].contiguous()
    exact, bound = lm.gated_recurrence(gs, xs), lm.gated_recurrence_bound(gs, xs)
    within(h[..., pick], exact[0], bound[0])
    within(last[:, pick], exact[2], bound[2])
    dg, dx, dh0 = ops.gated_recurrence_backward(gate, x, states, h)
    hs = h[..., pick].contiguous()
    for got, e, o in zip((dg[..., pick], dx[..., pick], dh0[:, pick]), lm.gated_recurrence_backward(gs, xs, None, hs),
                         lm.gated_recurrence_backward_bound(gs, xs, None, hs)):
        within(got, e, o)
