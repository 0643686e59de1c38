"""What the language-model operators refuse, checked before any launch (no GPU needed)."""
import pytest
import torch

from hfuse_b200 import _lib, ops

BAD, ALIGN, LARGE, WORK = -1, -2, -3, -4
P = 4096                      # an address that is never followed


def _ln(x=P, rows=2, D=8, ld=8, t=0, w=P, b=P, wt=0, eps=1e-5, y=P, m=P, r=P):
    return _lib.lib().hfuse_layernorm(x, rows, D, ld, t, w, b, wt, eps, y, m, r, None)


def _lnb(x=P, ldx=8, dy=P, ldy=8, rows=2, D=8, t=0, m=P, r=P, w=P, wt=0, dx=P, dw=P, db=P, ws=P, nb=1 << 30):
    return _lib.lib().hfuse_layernorm_backward(x, ldx, dy, ldy, rows, D, t, m, r, w, wt, dx, dw, db, ws, nb, None)


def _emb(table=P, rows=4, D=8, t=0, ids=P, n=2, ib=8, out=P):
    return _lib.lib().hfuse_embedding(table, rows, D, t, ids, n, ib, 1.0, out, None)


def _embb(dy=P, ids=P, n=2, ib=8, rows=4, D=8, t=0, g=P, ws=P, nb=1 << 30):
    return _lib.lib().hfuse_embedding_backward(dy, ids, n, ib, rows, D, t, 1.0, -1, g, ws, nb, None)


def _rec(g=P, gb=8, gt=8, x=P, xb=8, xt=8, B=1, T=1, D=8, t=0, h0=None, y=P, last=P, st=None):
    return _lib.lib().hfuse_gated_recurrence(g, gb, gt, x, xb, xt, B, T, D, t, h0, y, last, st, None)


def _recb(g=P, gb=8, gt=8, x=P, xb=8, xt=8, st=P, dy=P, yb=8, yt=8, dl=None, B=1, T=1, D=8, t=0, dg=P, dx=P, dh=P):
    return _lib.lib().hfuse_gated_recurrence_backward(g, gb, gt, x, xb, xt, st, dy, yb, yt, dl, B, T, D, t, dg, dx, dh, None)


@pytest.mark.parametrize("call,kw,code", [
    (_ln, dict(x=None), BAD), (_ln, dict(y=None), BAD), (_ln, dict(m=None), BAD), (_ln, dict(r=None), BAD), (_ln, dict(D=0), BAD),
    (_ln, dict(rows=-1), BAD), (_ln, dict(ld=7), BAD), (_ln, dict(t=3), BAD), (_ln, dict(t=0, wt=1), BAD), (_ln, dict(t=1, wt=2), BAD),
    (_ln, dict(eps=-1.0), BAD), (_ln, dict(eps=float("nan")), BAD), (_ln, dict(x=P + 2), ALIGN), (_ln, dict(w=P + 1, t=1, wt=1), ALIGN),
    (_ln, dict(m=P + 2), ALIGN), (_ln, dict(rows=0, x=None), 0), (_ln, dict(D=(1 << 30) + 1, ld=1 << 31), LARGE),
    (_lnb, dict(D=(1 << 30) + 1, ldx=1 << 31, ldy=1 << 31), LARGE), (_emb, dict(D=(1 << 30) + 1), LARGE), (_embb, dict(D=(1 << 30) + 1), LARGE),
    (_rec, dict(D=(1 << 30) + 1), LARGE), (_recb, dict(D=(1 << 30) + 1), LARGE),
    (_lnb, dict(x=None), BAD), (_lnb, dict(dy=None), BAD), (_lnb, dict(m=None), BAD), (_lnb, dict(ldx=7), BAD), (_lnb, dict(ldy=7), BAD),
    (_lnb, dict(D=-1), BAD), (_lnb, dict(t=5), BAD), (_lnb, dict(wt=1), BAD), (_lnb, dict(ws=None), WORK), (_lnb, dict(nb=8), WORK),
    (_lnb, dict(dx=P + 2), ALIGN), (_lnb, dict(ws=P + 8), ALIGN),
    (_emb, dict(table=None), BAD), (_emb, dict(ids=None), BAD), (_emb, dict(out=None), BAD), (_emb, dict(rows=0), BAD), (_emb, dict(D=0), BAD),
    (_emb, dict(n=-1), BAD), (_emb, dict(ib=2), BAD), (_emb, dict(t=9), BAD), (_emb, dict(rows=1 << 31), LARGE), (_emb, dict(n=1 << 31), LARGE),
    (_emb, dict(table=P + 2), ALIGN), (_emb, dict(ids=P + 4), ALIGN), (_emb, dict(n=0, ids=None), 0),
    (_embb, dict(dy=None), BAD), (_embb, dict(ids=None), BAD), (_embb, dict(g=None), BAD), (_embb, dict(ib=1), BAD), (_embb, dict(rows=0), BAD),
    (_embb, dict(rows=1 << 31), LARGE), (_embb, dict(n=1 << 31), LARGE), (_embb, dict(ws=None), WORK), (_embb, dict(nb=16), WORK),
    (_embb, dict(g=P + 1, t=1), ALIGN), (_embb, dict(ids=P + 4), ALIGN),
    (_rec, dict(g=None), BAD), (_rec, dict(x=None), BAD), (_rec, dict(y=None), BAD), (_rec, dict(last=None), BAD), (_rec, dict(B=0), BAD),
    (_rec, dict(T=0), BAD), (_rec, dict(D=0), BAD), (_rec, dict(gt=-8), BAD), (_rec, dict(t=4), BAD), (_rec, dict(T=1 << 31), LARGE),
    (_rec, dict(B=1 << 20, D=1 << 20), LARGE), (_rec, dict(x=P + 1, t=1), ALIGN), (_rec, dict(h0=P + 2), ALIGN),
    (_recb, dict(st=None), BAD), (_recb, dict(dy=None), BAD), (_recb, dict(dg=None), BAD), (_recb, dict(dx=None), BAD), (_recb, dict(dh=None), BAD),
    (_recb, dict(yt=-1), BAD), (_recb, dict(T=0), BAD), (_recb, dict(T=1 << 31), LARGE), (_recb, dict(st=P + 2), ALIGN),
])
def test_c_entry_points(call, kw, code):
    assert call(**kw) == code


def test_workspace_sizes():
    L = _lib.lib()
    assert L.hfuse_layernorm_backward_workspace_bytes(-1, 8) == 0 and L.hfuse_layernorm_backward_workspace_bytes(4, 0) == 0
    assert L.hfuse_layernorm_backward_workspace_bytes(0, 8) >= 64
    assert L.hfuse_embedding_backward_workspace_bytes(0, 8, 8) == 0 and L.hfuse_embedding_backward_workspace_bytes(1 << 31, 8, 8) == 0
    assert L.hfuse_embedding_backward_workspace_bytes(100, 8, 8) >= 100 * 16
    for T, chunks in ((0, 0), (1, 1), (256, 1), (257, 2), (1 << 20, 4096)):
        assert L.hfuse_gated_recurrence_chunks(T) == chunks


def test_python_entry_points_refuse_cpu_tensors():
    from hfuse_b200 import torch_ops  # noqa: F401
    T = torch.ops.hfuse_b200
    x, ids, z = torch.zeros(2, 4), torch.zeros(2, dtype=torch.int64), torch.zeros(2, 3, 4)
    row = torch.zeros(2)
    for call in (lambda: ops.layer_norm(x), lambda: T.layer_norm(x, None, None, 1e-5),
                 lambda: ops.layer_norm_backward(x, x, row, row), lambda: T.layer_norm_backward(x, x, row, row, None),
                 lambda: ops.embedding(x, ids), lambda: T.embedding(x, ids, 1.0),
                 lambda: ops.embedding_backward(x, ids, 4), lambda: T.embedding_backward(x, ids, 4, 1.0, -1),
                 lambda: ops.gated_recurrence(z, z), lambda: T.gated_recurrence(z, z, None, False),
                 lambda: ops.gated_recurrence_backward(z, z, z, z), lambda: T.gated_recurrence_backward(z, z, z, z, None)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(TypeError):
        ops.layer_norm([1.0])
