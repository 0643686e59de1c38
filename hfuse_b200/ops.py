"""Python call harness for the deep-learning kernels and their fused pairs.

Plays the part of the reference's `TorchKernel/call_{1080,v100}.py` harness
(README.md:84-95 of aoli-al/HFuse): it hands CUDA tensors to the fused entry
points.  PyTorch only supplies device memory and the current stream; every
operator below runs a hand-written sm_100a kernel through the C ABI, and
raises if the tensors are not on a CUDA device — there is no CPU path.

An operator is described by a small object (`Im2col`, `MaxPool`, `BnStats`,
`Upsample`, `Histc`) that owns its output buffers; `run(op)` launches the
standalone kernel, `run_pair(a, b)` launches the fused pair named after the
two halves (the ten pairs of the reference's configs/ml_fusion.yaml).

The operators of a language model's token path (`layer_norm`, `embedding`,
`gated_recurrence` and their backward functions) are plain functions that
allocate their results; gradients are explicit calls, as for pooling and batch norm.
"""
from __future__ import annotations

import torch

from . import _lib


def _check_input(x: torch.Tensor, name: str) -> torch.Tensor:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not x.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor: hfuse_b200 has no CPU path")
    if x.dtype != torch.float32:
        raise TypeError(f"{name} must be float32, got {x.dtype}")
    if not x.is_contiguous():
        raise ValueError(f"{name} must be contiguous (NCHW)")
    return x


def _pair(v):
    return (v, v) if isinstance(v, int) else tuple(v)


def _stream_ptr(stream=None) -> int:
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


class Im2col:
    """unfold: x [N,C,H,W] -> col [N, C*kh*kw, Hc*Wc]"""
    key = "im2col"

    def __init__(self, x, kernel_size, padding=0, stride=1, dilation=1, out=None):
        self.x = _check_input(x, "im2col input")
        if x.dim() != 4:
            raise ValueError("im2col input must be 4-D")
        (self.kh, self.kw), (self.ph, self.pw) = _pair(kernel_size), _pair(padding)
        (self.sh, self.sw), (self.dh, self.dw) = _pair(stride), _pair(dilation)
        N, C, H, W = x.shape
        Hc = (H + 2 * self.ph - (self.dh * (self.kh - 1) + 1)) // self.sh + 1
        Wc = (W + 2 * self.pw - (self.dw * (self.kw - 1) + 1)) // self.sw + 1
        if Hc <= 0 or Wc <= 0:
            raise ValueError("im2col: kernel does not fit the padded input")
        self.Hc, self.Wc = Hc, Wc
        self.out = out if out is not None else torch.empty(
            (N, C * self.kh * self.kw, Hc * Wc), dtype=torch.float32, device=x.device)

    def c_args(self):
        N, C, H, W = self.x.shape
        return [self.x.data_ptr(), N, C, H, W, self.kh, self.kw, self.ph, self.pw, self.sh, self.sw,
                self.dh, self.dw, self.out.data_ptr()]

    def result(self):
        return self.out


class MaxPool:
    """max_pool2d_with_indices: x [N,C,H,W] -> (values, int64 indices) [N,C,pH,pW]"""
    key = "maxpool"

    def __init__(self, x, kernel_size, stride=None, padding=0, dilation=1, out=None, indices=None):
        self.x = _check_input(x, "max_pool input")
        if x.dim() != 4:
            raise ValueError("max_pool input must be 4-D")
        (self.kh, self.kw) = _pair(kernel_size)
        (self.sh, self.sw) = _pair(stride) if stride is not None else (self.kh, self.kw)
        (self.ph, self.pw), (self.dh, self.dw) = _pair(padding), _pair(dilation)
        N, C, H, W = x.shape
        self.pH = (H + 2 * self.ph - self.dh * (self.kh - 1) - 1) // self.sh + 1
        self.pW = (W + 2 * self.pw - self.dw * (self.kw - 1) - 1) // self.sw + 1
        if self.pH <= 0 or self.pW <= 0:
            raise ValueError("max_pool: window does not fit the padded input")
        shape = (N, C, self.pH, self.pW)
        self.out = out if out is not None else torch.empty(shape, dtype=torch.float32, device=x.device)
        self.idx = indices if indices is not None else torch.empty(shape, dtype=torch.int64, device=x.device)

    def c_args(self):
        N, C, H, W = self.x.shape
        return [self.x.data_ptr(), N, C, H, W, self.pH, self.pW, self.kh, self.kw, self.sh, self.sw,
                self.ph, self.pw, self.dh, self.dw, self.out.data_ptr(), self.idx.data_ptr()]

    def result(self):
        return self.out, self.idx


_workspaces: dict = {}


def bn_workspace(C: int, device) -> torch.Tensor:
    """Zero-initialised scratch for the statistics kernel, one per (device, stream, C)."""
    key = (str(device), torch.cuda.current_stream(device).cuda_stream, C)
    ws = _workspaces.get(key)
    if ws is None:
        nbytes = _lib.lib().hfuse_bnstats_workspace_bytes(1, C, 1)
        ws = torch.zeros(nbytes, dtype=torch.uint8, device=device)
        _workspaces[key] = ws
    return ws


class BnStats:
    """batch_norm_collect_statistics: x [N,C,...] -> (mean[C], invstd[C]); optional fp64 moments [C,3]"""
    key = "bnstats"

    def __init__(self, x, eps=1e-5, want_moments=False, workspace=None):
        self.x = _check_input(x, "batch_norm input")
        if x.dim() < 2:
            raise ValueError("batch_norm input must have at least 2 dimensions")
        self.N, self.C = x.shape[0], x.shape[1]
        self.HW = x.numel() // (self.N * self.C) if self.N * self.C else 0
        self.eps = float(eps)
        self.mean = torch.empty(self.C, dtype=torch.float32, device=x.device)
        self.invstd = torch.empty(self.C, dtype=torch.float32, device=x.device)
        self.moments = torch.empty((self.C, 3), dtype=torch.float64, device=x.device) if want_moments else None
        self.ws = workspace if workspace is not None else bn_workspace(self.C, x.device)

    def c_args(self):
        return [self.x.data_ptr(), self.N, self.C, self.HW, self.eps, self.mean.data_ptr(),
                self.invstd.data_ptr(), self.moments.data_ptr() if self.moments is not None else None,
                self.ws.data_ptr(), self.ws.numel()]

    def result(self):
        return self.mean, self.invstd


class Upsample:
    """upsample_bilinear2d: x [N,C,H,W] -> [N,C,outH,outW]"""
    key = "upsample"

    def __init__(self, x, size=None, scale_factor=None, align_corners=False, out=None):
        self.x = _check_input(x, "upsample input")
        if x.dim() != 4:
            raise ValueError("upsample input must be 4-D")
        N, C, H, W = x.shape
        if size is None:
            if scale_factor is None:
                raise ValueError("give size or scale_factor")
            sh, sw = (scale_factor, scale_factor) if not isinstance(scale_factor, (tuple, list)) else scale_factor
            size = (int(H * sh), int(W * sw))
        self.outH, self.outW = _pair(size)
        if self.outH <= 0 or self.outW <= 0:
            raise ValueError("upsample: output size must be positive")
        self.align = bool(align_corners)
        self.out = out if out is not None else torch.empty((N, C, self.outH, self.outW), dtype=torch.float32,
                                                           device=x.device)

    def c_args(self):
        N, C, H, W = self.x.shape
        return [self.x.data_ptr(), N, C, H, W, self.outH, self.outW, int(self.align), self.out.data_ptr()]

    def result(self):
        return self.out


class Histc:
    """histc: all elements of x -> uint32 counts[bins] over [min, max] (stored as int32 bits in torch)"""
    key = "histc"

    def __init__(self, x, bins=100, min=0.0, max=0.0, out=None):
        self.x = _check_input(x, "histc input")
        if bins <= 0:
            raise ValueError("histc: bins must be positive")
        if float(min) == float(max):
            # same rule as torch.histc: derive the range from the data
            if x.numel():
                lo, hi = float(x.min()), float(x.max())
            else:
                lo, hi = 0.0, 0.0
            if lo == hi:
                lo, hi = lo - 1.0, hi + 1.0
            min, max = lo, hi
        if not float(min) < float(max):
            raise ValueError("histc: max must be larger than min")
        self.bins, self.lo, self.hi = int(bins), float(min), float(max)
        self.counts = out if out is not None else torch.empty(self.bins, dtype=torch.int32, device=x.device)

    def c_args(self):
        return [self.x.data_ptr(), self.x.numel(), self.bins, self.lo, self.hi, self.counts.data_ptr()]

    def result(self):
        return self.counts


def run(op, stream=None):
    """Launch the standalone kernel of one operator on the current (or given) stream."""
    fn = getattr(_lib.lib(), _lib.DL_SOLO[op.key])
    _lib.check(fn(*op.c_args(), _stream_ptr(stream)), _lib.DL_SOLO[op.key])
    return op.result()


def pair_name(a, b) -> str:
    name = f"{a.key}_{b.key}"
    if name not in _lib.DL_PAIRS:
        raise KeyError(f"no fused pair {name}; the pairs are {sorted(_lib.DL_PAIRS)}")
    return name


def run_pair(a, b, stream=None):
    """Launch the fused pair (a, b) as ONE kernel."""
    name = pair_name(a, b)
    fn = getattr(_lib.lib(), f"hfuse_{name}_f32")
    _lib.check(fn(*a.c_args(), *b.c_args(), _stream_ptr(stream)), f"hfuse_{name}_f32")
    return a.result(), b.result()


def run_back_to_back(a, b, stream=None):
    """The unfused baseline: the two standalone kernels queued on one stream with no
    host synchronisation in between (the reference's "ST" measurement,
    scripts/analyze_nvprof.py:264-284)."""
    return run(a, stream), run(b, stream)


# ---- functional conveniences, named after the torch operators they stand in for --------
def im2col(x, kernel_size, padding=0, stride=1, dilation=1):
    return run(Im2col(x, kernel_size, padding, stride, dilation))


def max_pool2d_with_indices(x, kernel_size, stride=None, padding=0, dilation=1):
    return run(MaxPool(x, kernel_size, stride, padding, dilation))


def batch_norm_stats(x, eps=1e-5):
    return run(BnStats(x, eps))


def upsample_bilinear2d(x, size=None, scale_factor=None, align_corners=False):
    return run(Upsample(x, size, scale_factor, align_corners))


def histc(x, bins=100, min=0.0, max=0.0):
    return run(Histc(x, bins, min, max))


def bn_finalize(moments: torch.Tensor, eps: float):
    """mean / invstd from fp64 moments [C,3] that were summed over GPUs."""
    if not moments.is_cuda or moments.dtype != torch.float64 or not moments.is_contiguous():
        raise ValueError("moments must be a contiguous CUDA float64 tensor [C,3]")
    Cn = moments.shape[0]
    mean = torch.empty(Cn, dtype=torch.float32, device=moments.device)
    invstd = torch.empty(Cn, dtype=torch.float32, device=moments.device)
    _lib.check(_lib.lib().hfuse_bnstats_finalize_f64(moments.data_ptr(), Cn, float(eps), mean.data_ptr(),
                                                     invstd.data_ptr(), _stream_ptr()),
               "hfuse_bnstats_finalize_f64")
    return mean, invstd


# ---- backward kernels (listed by the reference next to the forward ones, never fused there) ------
class MaxPoolBackward:
    """grad_in of max_pool2d from grad_out and the indices a MaxPool operator wrote."""

    def __init__(self, fwd: MaxPool, grad_out: torch.Tensor):
        self.fwd = fwd
        self.grad_out = _check_input(grad_out, "max_pool grad_out")
        if tuple(grad_out.shape) != tuple(fwd.out.shape):
            raise ValueError("grad_out must have the shape of the pooled output")
        self.grad_in = torch.empty_like(fwd.x)

    def c_args(self):
        f = self.fwd
        N, C, H, W = f.x.shape
        return [self.grad_out.data_ptr(), f.idx.data_ptr(), N, C, H, W, f.pH, f.pW, f.kh, f.kw, f.sh, f.sw, f.ph, f.pw,
                f.dh, f.dw, self.grad_in.data_ptr()]


class BnBackward:
    """Training-mode batch-norm backward from the saved mean / invstd of the statistics kernel."""

    def __init__(self, x, grad_out, mean, invstd, weight=None):
        self.x, self.dy = _check_input(x, "batch_norm input"), _check_input(grad_out, "batch_norm grad_out")
        if x.shape != grad_out.shape:
            raise ValueError("grad_out must have the shape of the input")
        self.N, self.C = x.shape[0], x.shape[1]
        self.HW = x.numel() // (self.N * self.C)
        self.mean, self.invstd, self.weight = mean, invstd, weight
        self.dx = torch.empty_like(x)
        self.grad_weight = torch.empty(self.C, dtype=torch.float32, device=x.device)
        self.grad_bias = torch.empty(self.C, dtype=torch.float32, device=x.device)

    def c_args(self):
        return [self.x.data_ptr(), self.dy.data_ptr(), self.N, self.C, self.HW,
                self.weight.data_ptr() if self.weight is not None else None, self.mean.data_ptr(),
                self.invstd.data_ptr(), self.dx.data_ptr(), self.grad_weight.data_ptr(), self.grad_bias.data_ptr()]


def max_pool2d_backward(fwd: MaxPool, grad_out, stream=None):
    op = MaxPoolBackward(fwd, grad_out)
    _lib.check(_lib.lib().hfuse_maxpool2d_backward_f32(*op.c_args(), _stream_ptr(stream)), "hfuse_maxpool2d_backward_f32")
    return op.grad_in


def batch_norm_backward(x, grad_out, mean, invstd, weight=None, stream=None):
    op = BnBackward(x, grad_out, mean, invstd, weight)
    _lib.check(_lib.lib().hfuse_bn_backward_f32(*op.c_args(), _stream_ptr(stream)), "hfuse_bn_backward_f32")
    return op.dx, op.grad_weight, op.grad_bias


def run_backward_pair(mp: MaxPoolBackward, bn: BnBackward, stream=None):
    """max-pool backward and batch-norm backward in ONE fused launch."""
    _lib.check(_lib.lib().hfuse_maxpool_backward_bn_backward_f32(*mp.c_args(), *bn.c_args(), _stream_ptr(stream)),
               "hfuse_maxpool_backward_bn_backward_f32")
    return mp.grad_in, (bn.dx, bn.grad_weight, bn.grad_bias)


# ---- operators of a language model's token path (forward and backward; f32, bf16 and f16) ----------
_LM_TYPES = {torch.float32: _lib.HFUSE_F32, torch.bfloat16: _lib.HFUSE_BF16, torch.float16: _lib.HFUSE_F16}


def _check_lm(x, name, dim=None, dtypes=None, shape=None, like=None):
    """Argument checks shared by the language-model operators; the innermost dimension has stride 1."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not x.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor: hfuse_b200 has no CPU path")
    if x.dtype not in (dtypes or _LM_TYPES):
        raise TypeError(f"{name} must be {' or '.join(str(t)[6:] for t in (dtypes or _LM_TYPES))}, got {x.dtype}")
    if like is not None and x.device != like.device:
        raise ValueError(f"{name} must be on {like.device}, is on {x.device}")
    if dim is not None and x.dim() != dim:
        raise ValueError(f"{name} must be {dim}-D")
    if shape is not None and tuple(x.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, has {tuple(x.shape)}")
    if x.dim() and x.shape[-1] > 1 and x.stride(-1) != 1:
        raise ValueError(f"{name} must have stride 1 in its last dimension")
    return x


def _row_length(x, name):
    """Elements of a row; the C entry points take a 32-bit number, of which ctypes would pass the lower bits."""
    if x.shape[-1] > 0x7fffffff:
        raise ValueError(f"{name} has too long rows")
    return x.shape[-1]


def _contiguous(x, name):
    if not x.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return x


def _row_stride(x, name):
    """Elements between two rows (all dimensions but the last one, which must follow each other evenly)."""
    ld, span = None, None
    if x.numel() == 0:
        return x.shape[-1]
    for d in range(x.dim() - 2, -1, -1):
        if x.shape[d] == 1:
            continue
        if ld is None:
            ld = x.stride(d)
        elif x.stride(d) != span:
            raise ValueError(f"{name} must have rows that are evenly spaced in memory")
        span = x.stride(d) * x.shape[d]
    if ld is None:
        return x.shape[-1]
    if ld < x.shape[-1]:
        raise ValueError(f"{name} must have rows that do not overlap")
    return ld


def _ptr(x):
    return None if x is None else x.data_ptr()


class _on:
    """Device and stream of a call: buffers made inside belong to the stream that the kernels run on."""

    def __init__(self, x, stream):
        if stream is not None and stream.device != x.device:
            raise ValueError(f"the stream must be one of {x.device}, is one of {stream.device}")
        self.stream = stream if stream is not None else torch.cuda.current_stream(x.device)

    def __enter__(self):
        self.ctx = torch.cuda.stream(self.stream)
        self.ctx.__enter__()
        return self.stream.cuda_stream

    def __exit__(self, *exc):
        return self.ctx.__exit__(*exc)


def _check_norm_params(x, weight, bias):
    D = x.shape[-1]
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            _contiguous(_check_lm(t, name, dtypes=(x.dtype, torch.float32), shape=(D,), like=x), name)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("weight and bias must have the same type")
    given = weight if weight is not None else bias
    return x.dtype if given is None else given.dtype


def layer_norm(x, weight=None, bias=None, eps=1e-5, stream=None):
    """x [..., D] -> (y [..., D], mean [...], invstd [...]); mean and invstd are float32."""
    _check_lm(x, "layer_norm input")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("layer_norm input must have a last dimension of at least 1")
    if not eps >= 0:
        raise ValueError("layer_norm: eps must not be negative")
    wt = _check_norm_params(x, weight, bias)
    D, ld = _row_length(x, "layer_norm input"), _row_stride(x, "layer_norm input")
    with _on(x, stream) as s:
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        mean = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
        invstd = torch.empty_like(mean)
        _lib.check(_lib.lib().hfuse_layernorm(x.data_ptr(), x.numel() // D, D, ld, _LM_TYPES[x.dtype], _ptr(weight), _ptr(bias),
                                              _LM_TYPES[wt], float(eps), y.data_ptr(), mean.data_ptr(), invstd.data_ptr(), s),
                   "hfuse_layernorm")
    return y, mean, invstd


def layer_norm_backward(x, grad_out, mean, invstd, weight=None, stream=None):
    """Gradients (grad_in, grad_weight, grad_bias) of layer_norm from what it saved.  grad_weight and grad_bias have
    the weight's type (the input's without a weight)."""
    _check_lm(x, "layer_norm input")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("layer_norm input must have a last dimension of at least 1")
    _check_lm(grad_out, "layer_norm grad_out", dtypes=(x.dtype,), shape=x.shape, like=x)
    for t, name in ((mean, "mean"), (invstd, "invstd")):
        _contiguous(_check_lm(t, name, dtypes=(torch.float32,), shape=x.shape[:-1], like=x), name)
    wt = _check_norm_params(x, weight, None)
    D = _row_length(x, "layer_norm input")
    rows = x.numel() // D
    ldx, ldg = _row_stride(x, "layer_norm input"), _row_stride(grad_out, "layer_norm grad_out")
    L = _lib.lib()
    with _on(x, stream) as s:
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dw, db = (torch.empty(D, dtype=wt, device=x.device) for _ in range(2))
        ws = torch.empty(L.hfuse_layernorm_backward_workspace_bytes(rows, D), dtype=torch.uint8, device=x.device)
        _lib.check(L.hfuse_layernorm_backward(x.data_ptr(), ldx, grad_out.data_ptr(), ldg, rows, D, _LM_TYPES[x.dtype],
                                              mean.data_ptr(), invstd.data_ptr(), _ptr(weight), _LM_TYPES[wt], dx.data_ptr(),
                                              dw.data_ptr(), db.data_ptr(), ws.data_ptr(), ws.numel(), s),
                   "hfuse_layernorm_backward")
    return dx, dw, db


def _check_ids(ids, like):
    return _contiguous(_check_lm(ids, "ids", dtypes=(torch.int64, torch.int32), like=like), "ids")


def embedding(table, ids, scale=1.0, stream=None):
    """scale * table[ids]: table [rows, D], ids of any shape (int64 or int32) -> ids.shape + [D]; an id outside the
    table gives zeros."""
    _contiguous(_check_lm(table, "embedding table", dim=2), "embedding table")
    if 0 in table.shape:
        raise ValueError("embedding table must not be empty")
    _check_ids(ids, table)
    rows, D = table.shape[0], _row_length(table, "embedding table")
    with _on(table, stream) as s:
        out = torch.empty(tuple(ids.shape) + (D,), dtype=table.dtype, device=table.device)
        _lib.check(_lib.lib().hfuse_embedding(table.data_ptr(), rows, D, _LM_TYPES[table.dtype], ids.data_ptr(), ids.numel(),
                                              ids.element_size(), float(scale), out.data_ptr(), s), "hfuse_embedding")
    return out


def embedding_backward(grad_out, ids, rows, scale=1.0, padding_id=-1, stream=None):
    """Gradient [rows, D] of embedding's table; ids outside [0, rows) and padding_id (-1: none) give none."""
    _contiguous(_check_lm(grad_out, "embedding grad_out"), "embedding grad_out")
    _check_ids(ids, grad_out)
    if grad_out.dim() < 1 or grad_out.shape[-1] < 1 or tuple(grad_out.shape[:-1]) != tuple(ids.shape):
        raise ValueError("embedding grad_out must have the shape of ids and one dimension more")
    if rows < 1:
        raise ValueError("embedding_backward: rows must be positive")
    D, n, L = _row_length(grad_out, "embedding grad_out"), ids.numel(), _lib.lib()
    with _on(grad_out, stream) as s:
        grad = torch.empty(rows, D, dtype=grad_out.dtype, device=grad_out.device)
        ws = torch.empty(L.hfuse_embedding_backward_workspace_bytes(n, rows, D), dtype=torch.uint8, device=grad_out.device)
        _lib.check(L.hfuse_embedding_backward(grad_out.data_ptr(), ids.data_ptr(), n, ids.element_size(), rows, D,
                                              _LM_TYPES[grad_out.dtype], float(scale), int(padding_id), grad.data_ptr(),
                                              ws.data_ptr(), ws.numel(), s), "hfuse_embedding_backward")
    return grad


def _check_steps(x, name, like=None):
    _check_lm(x, name, dim=3, dtypes=None if like is None else (like.dtype,), shape=None if like is None else like.shape, like=like)
    if 0 in x.shape:
        raise ValueError(f"{name} must not be empty")
    _row_length(x, name)
    return x


def _check_state(h, name, x):
    if h is not None:
        _contiguous(_check_lm(h, name, dtypes=(torch.float32,), shape=(x.shape[0], x.shape[2]), like=x), name)
    return h


def gated_recurrence(gate, x, h0=None, save_states=False, stream=None):
    """h_t = sigmoid(gate_t) h_{t-1} + (1 - sigmoid(gate_t)) x_t along dimension 1 of gate, x [B, T, D] ->
    (h [B, T, D], the last state [B, D] in float32, states for gated_recurrence_backward or an empty tensor)."""
    _check_steps(gate, "gate")
    _check_steps(x, "x", gate)
    _check_state(h0, "h0", x)
    B, T, D = x.shape
    L = _lib.lib()
    with _on(x, stream) as s:
        out = torch.empty((B, T, D), dtype=x.dtype, device=x.device)
        last = torch.empty((B, D), dtype=torch.float32, device=x.device)
        states = torch.empty((B, L.hfuse_gated_recurrence_chunks(T), D) if save_states else (0,), dtype=torch.float32,
                             device=x.device)
        _lib.check(L.hfuse_gated_recurrence(gate.data_ptr(), gate.stride(0), gate.stride(1), x.data_ptr(), x.stride(0),
                                            x.stride(1), B, T, D, _LM_TYPES[x.dtype], _ptr(h0), out.data_ptr(), last.data_ptr(),
                                            states.data_ptr() if save_states else None, s), "hfuse_gated_recurrence")
    return out, last, states


def gated_recurrence_backward(gate, x, states, grad_out, grad_last=None, stream=None):
    """Gradients (grad_gate, grad_x, grad_h0) of gated_recurrence from the states that it saved; grad_last [B, D] is the
    gradient of the last state."""
    _check_steps(gate, "gate")
    _check_steps(x, "x", gate)
    _check_steps(grad_out, "grad_out", gate)
    _check_state(grad_last, "grad_last", x)
    B, T, D = x.shape
    L = _lib.lib()
    _contiguous(_check_lm(states, "states", dtypes=(torch.float32,), shape=(B, L.hfuse_gated_recurrence_chunks(T), D), like=x),
                "states")
    with _on(x, stream) as s:
        dgate, dx = (torch.empty((B, T, D), dtype=x.dtype, device=x.device) for _ in range(2))
        dh0 = torch.empty((B, D), dtype=torch.float32, device=x.device)
        _lib.check(L.hfuse_gated_recurrence_backward(
            gate.data_ptr(), gate.stride(0), gate.stride(1), x.data_ptr(), x.stride(0), x.stride(1), states.data_ptr(),
            grad_out.data_ptr(), grad_out.stride(0), grad_out.stride(1), _ptr(grad_last), B, T, D, _LM_TYPES[x.dtype],
            dgate.data_ptr(), dx.data_ptr(), dh0.data_ptr(), s), "hfuse_gated_recurrence_backward")
    return dgate, dx, dh0
