"""Cases of the language-model operators: layer norm, scaled embedding lookup with its gradient, gated linear recurrence.

Every case can be run in two forms that take the same inputs: `own = True` calls the library's operators
(torch.ops.hfuse_b200.*), `own = False` computes the same values with elementary torch operations in 32 bits, rounded
once at the end.  `exact` is the definition in 64 bits.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CHUNK = 256          # steps between two states that the recurrence's forward pass saves for its backward pass
EPS = 1e-5


def listed():
    return [
        # a decoding step normalises one token's activations: launch latency and nothing else
        {"name": "layer_norm_one_row", "op": "layer_norm", "way": "forward", "type": "bf16", "wtype": "bf16", "rows": 1, "dim": 4096},
        # a training batch of 8 sequences of 2048 tokens, half precision throughout
        {"name": "layer_norm_batch", "op": "layer_norm", "way": "forward", "type": "bf16", "wtype": "bf16", "rows": 16384, "dim": 4096},
        # its backward pass in a full-precision model of half the width
        {"name": "layer_norm_grad_f32", "op": "layer_norm", "way": "backward", "type": "f32", "wtype": "f32", "rows": 8192, "dim": 2048},
        # an odd width, a ragged number of tokens, half-precision activations under full-precision weights
        {"name": "layer_norm_grad_odd", "op": "layer_norm", "way": "backward", "type": "f16", "wtype": "f32", "rows": 12345, "dim": 1001},
        # the lookup of a decoding step for 32 sequences
        {"name": "embedding_decode", "op": "embedding", "way": "forward", "type": "bf16", "tokens": 32, "dim": 4096, "vocab": 32000},
        # the lookup of a training batch
        {"name": "embedding_batch", "op": "embedding", "way": "forward", "type": "f32", "tokens": 16384, "dim": 2048, "vocab": 50257},
        # the gradient of a small ragged batch with an odd width: most rows of the table are not met
        {"name": "embedding_grad_small", "op": "embedding", "way": "backward", "type": "f16", "tokens": 4099, "dim": 1001, "vocab": 32000},
        # the gradient of a large batch over a large vocabulary, token frequencies as in text
        {"name": "embedding_grad_batch", "op": "embedding", "way": "backward", "type": "bf16", "tokens": 65536, "dim": 2048, "vocab": 128000},
        # one generated token for 64 sequences: the state is read, moved on and written
        {"name": "recurrence_step", "op": "recurrence", "way": "forward", "type": "bf16", "batch": 64, "steps": 1, "dim": 2048, "h0": True},
        # a training batch
        {"name": "recurrence_batch", "op": "recurrence", "way": "forward", "type": "bf16", "batch": 8, "steps": 4096, "dim": 2048, "h0": False},
        # one long document of odd length, few channels: the scan itself has to be split
        {"name": "recurrence_long", "op": "recurrence", "way": "forward", "type": "f32", "batch": 1, "steps": 65537, "dim": 768, "h0": True},
        # the backward pass of a training batch
        {"name": "recurrence_grad", "op": "recurrence", "way": "backward", "type": "bf16", "batch": 4, "steps": 8192, "dim": 1024, "h0": True},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A model width: two out of three are multiples of 64 (or 8 where small), the others are anything."""
    d = _spread(rng, lo, hi)
    return d if rng.random() < 1 / 3 else max(lo, d // 64 * 64 if d >= 64 else d // 8 * 8)


def draw(rng):
    op = rng.choice(["layer_norm", "embedding", "recurrence"])
    kind = rng.choice(["f32", "bf16", "f16"])
    way = rng.choice(["forward", "backward"])
    if op == "layer_norm":
        dim = _width(rng, 32, 8192)
        rows = _spread(rng, 1, max(1, min(32768, (1 << 25) // dim)))
        return {"op": op, "way": way, "type": kind, "wtype": rng.choice([kind, "f32"]), "rows": rows, "dim": dim}
    if op == "embedding":
        dim = _width(rng, 32, 4096)
        vocab = _spread(rng, 100, max(100, min(200000, (1 << 27) // dim)))
        tokens = _spread(rng, 1, max(1, min(65536, (1 << 26) // dim)))
        return {"op": op, "way": way, "type": kind, "tokens": tokens, "dim": dim, "vocab": vocab}
    dim = _width(rng, 32, 4096)
    batch = _spread(rng, 1, 64)
    steps = _spread(rng, 1, max(1, min(65536, (1 << 25) // (dim * batch))))
    return {"op": op, "way": way, "type": kind, "batch": batch, "steps": steps, "dim": dim, "h0": rng.random() < 0.5}


# ---- the definitions in elementary operations -------------------------------------------------------------------
def _plain_layer_norm(x, weight, bias):
    f = x.float()
    mean = f.mean(-1, keepdim=True)
    d = f - mean
    invstd = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + EPS)
    y = d * invstd * weight.float() + bias.float()
    return y.to(x.dtype), mean.squeeze(-1), invstd.squeeze(-1)


def _plain_layer_norm_backward(x, grad_out, mean, invstd, weight):
    dy, r = grad_out.float(), invstd.unsqueeze(-1)
    xh = (x.float() - mean.unsqueeze(-1)) * r
    g = dy * weight.float()
    dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return dx.to(x.dtype), (dy * xh).sum(0).to(weight.dtype), dy.sum(0).to(weight.dtype)


def _plain_embedding(table, ids, scale):
    return (table[ids].float() * scale).to(table.dtype)


def _plain_embedding_backward(grad_out, ids, rows, scale):
    g = torch.zeros(rows, grad_out.shape[-1], dtype=torch.float32, device=grad_out.device)
    g.index_add_(0, ids, grad_out.float())
    return (g * scale).to(grad_out.dtype)


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1 by doubling the span that each step covers (a step by itself would
    be one launch for every token)."""
    a, b, s = a.clone(), b.clone(), 1
    while s < b.shape[1]:
        b[:, s:] = b[:, s:] + a[:, s:] * b[:, :-s]
        a[:, s:] = a[:, s:] * a[:, :-s]
        s *= 2
    return a, b


def _hidden(gate, x, h0, wide=torch.float32):
    a = torch.sigmoid(gate.to(wide))
    p, h = _scan(a, torch.sigmoid(-gate.to(wide)) * x.to(wide))
    return h if h0 is None else h + p * h0.to(wide).unsqueeze(1)


def _plain_recurrence(gate, x, h0):
    h = _hidden(gate, x, h0)
    return h.to(x.dtype), h[:, -1].contiguous()


def _plain_recurrence_backward(gate, x, states, grad_out, grad_last):
    h0 = states[:, 0]
    h = _hidden(gate, x, h0)
    before = torch.cat([h0.unsqueeze(1), h[:, :-1]], 1)
    a, z = torch.sigmoid(gate.float()), torch.sigmoid(-gate.float())
    d = grad_out.float()
    d[:, -1] += grad_last
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    e = _scan(later.flip(1), d.flip(1))[1].flip(1)
    return (e * (before - x.float()) * a * z).to(gate.dtype), (e * z).to(x.dtype), a[:, 0] * e[:, 0]


# ---- inputs --------------------------------------------------------------------------------------------------------
def _words(n, vocab, gen, dev):
    """Token ids with the frequencies of text (the k-th commonest word is met 1/k as often), the common ones spread
    over the vocabulary."""
    u = torch.rand(n, generator=gen, device=dev, dtype=torch.float64)
    rank = (torch.exp(u * math.log(vocab + 1.0)) - 1.0).long().clamp_(0, vocab - 1)
    return torch.randperm(vocab, generator=gen, device=dev)[rank]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    kind = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    s = dict(case)
    if case["op"] == "layer_norm":
        wt, D = TYPES[case["wtype"]], case["dim"]
        s["x"] = (0.3 + normal(case["rows"], D) * (0.5 + torch.rand(case["rows"], 1, generator=gen, device=dev))).to(kind)
        s["weight"], s["bias"] = (1 + 0.1 * normal(D)).to(wt), (0.1 * normal(D)).to(wt)
        if case["way"] == "backward":
            s["grad_out"] = normal(case["rows"], D).to(kind)
            wide = s["x"].double()
            s["mean"] = wide.mean(-1).float()
            s["invstd"] = (wide.var(-1, unbiased=False) + EPS).rsqrt().float()
    elif case["op"] == "embedding":
        s["ids"] = _words(case["tokens"], case["vocab"], gen, dev)
        s["scale"] = math.sqrt(case["dim"])
        if case["way"] == "forward":
            s["table"] = (normal(case["vocab"], case["dim"]) * 0.02).to(kind)
        else:
            s["grad_out"] = (normal(case["tokens"], case["dim"]) * 0.1).to(kind)
    else:
        shape = (case["batch"], case["steps"], case["dim"])
        s["gate"], s["x"] = (2 + 2 * normal(*shape)).to(kind), normal(*shape).to(kind)
        s["start"] = normal(case["batch"], case["dim"]) if case["h0"] else None
        if case["way"] == "backward":
            first = s["start"] if case["h0"] else torch.zeros(case["batch"], case["dim"], device=dev)
            h = _hidden(s["gate"], s["x"], first, torch.float64)
            s["states"] = torch.cat([first.unsqueeze(1), h[:, CHUNK - 1:-1:CHUNK].float()], 1).contiguous()
            s["grad_out"] = normal(*shape).to(kind)
            s["grad_last"] = normal(case["batch"], case["dim"])
    return s


def run(s):
    forward = s["way"] == "forward"
    if own:
        from hfuse_b200.torch_ops import ops
        if s["op"] == "layer_norm":
            if forward:
                return ops.layer_norm(s["x"], s["weight"], s["bias"], EPS)
            return ops.layer_norm_backward(s["x"], s["grad_out"], s["mean"], s["invstd"], s["weight"])
        if s["op"] == "embedding":
            if forward:
                return ops.embedding(s["table"], s["ids"], s["scale"])
            return ops.embedding_backward(s["grad_out"], s["ids"], s["vocab"], s["scale"], -1)
        if forward:
            return ops.gated_recurrence(s["gate"], s["x"], s["start"], False)[:2]
        return ops.gated_recurrence_backward(s["gate"], s["x"], s["states"], s["grad_out"], s["grad_last"])
    if s["op"] == "layer_norm":
        if forward:
            return _plain_layer_norm(s["x"], s["weight"], s["bias"])
        return _plain_layer_norm_backward(s["x"], s["grad_out"], s["mean"], s["invstd"], s["weight"])
    if s["op"] == "embedding":
        if forward:
            return _plain_embedding(s["table"], s["ids"], s["scale"])
        return _plain_embedding_backward(s["grad_out"], s["ids"], s["vocab"], s["scale"])
    if forward:
        return _plain_recurrence(s["gate"], s["x"], s["start"])
    return _plain_recurrence_backward(s["gate"], s["x"], s["states"], s["grad_out"], s["grad_last"])


def work(case):
    e, D = (4 if case["type"] == "f32" else 2), case["dim"]
    forward = case["way"] == "forward"
    if case["op"] == "layer_norm":
        we, n = (4 if case["wtype"] == "f32" else 2), case["rows"] * D
        if forward:
            return {"bytes": 2 * n * e + 8 * case["rows"] + 2 * D * we, "flops": 8 * n}
        return {"bytes": 3 * n * e + 8 * case["rows"] + 3 * D * we, "flops": 14 * n}
    if case["op"] == "embedding":
        n, V = case["tokens"], case["vocab"]
        if forward:
            # rows of the table that n tokens with these frequencies are expected to meet
            top = math.log(V + 1.0)
            met, k = 0.0, 0
            while k < V:
                m = max(1, k // 50)
                share = min(1.0, (math.log(min(V, k + m) + 1.0) - math.log(k + 1.0)) / top / m)
                met += min(m, V - k) * -math.expm1(n * math.log1p(-share)) if share < 1 else min(m, V - k)
                k += m
            return {"bytes": (n + met) * D * e + 8 * n, "flops": n * D}
        return {"bytes": (n + V) * D * e + 8 * n, "flops": 2 * n * D}
    n, bd = case["batch"] * case["steps"] * D, case["batch"] * D
    if forward:
        return {"bytes": 3 * n * e + (8 if case["h0"] else 4) * bd, "flops": 8 * n}
    chunks = -(-case["steps"] // CHUNK)
    return {"bytes": 5 * n * e + 4 * bd * (2 + chunks), "flops": 20 * n}


# ---- the definitions in 64 bits, step by step ------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "layer_norm":
        x, w = s["x"].double(), s["weight"].double()
        D = x.shape[1]
        if case["way"] == "forward":
            mean = torch.einsum("rd->r", x) / D
            var = torch.einsum("rd,rd->r", x, x) / D - mean ** 2
            r = (var + EPS) ** -0.5
            return torch.addcmul(s["bias"].double(), (x - mean[:, None]) * r[:, None], w), mean, r
        r, dy = s["invstd"].double()[:, None], s["grad_out"].double()
        xh = r * x - r * s["mean"].double()[:, None]
        # dx = r (I - 1 1'/D - xh xh'/D) (w dy)
        along = torch.einsum("rd,rd,d->r", dy, xh, w)[:, None]
        dx = r / D * (D * dy * w - torch.einsum("rd,d->r", dy, w)[:, None] - xh * along)
        return dx, torch.einsum("rd,rd->d", dy, xh), torch.einsum("rd->d", dy)
    if case["op"] == "embedding":
        if case["way"] == "forward":
            return torch.nn.functional.embedding(s["ids"], s["table"]).double() * s["scale"]
        g = torch.zeros(case["vocab"], case["dim"], dtype=torch.float64, device=s["ids"].device)
        for at in range(0, case["tokens"], 4096):
            part = s["grad_out"][at:at + 4096].double() * s["scale"]
            g.index_put_((s["ids"][at:at + 4096],), part, accumulate=True)
        return g
    if case["steps"] > 70000:
        return None
    first = s["start"] if case["way"] == "forward" else s["states"][:, 0]
    h = first.double() if first is not None else torch.zeros(case["batch"], case["dim"], dtype=torch.float64, device="cuda")
    g, x = s["gate"].double(), s["x"].double()
    a = 1 / (1 + torch.exp(-g))
    every = torch.empty_like(x)
    for t in range(case["steps"]):
        if case["way"] == "backward":
            every[:, t] = h
        h = x[:, t] + a[:, t] * (h - x[:, t])
        if case["way"] == "forward":
            every[:, t] = h
    if case["way"] == "forward":
        return every, h
    e = s["grad_last"].double()
    dg, dx, dy = torch.empty_like(x), torch.empty_like(x), s["grad_out"].double()
    for t in range(case["steps"] - 1, -1, -1):
        e = e + dy[:, t]
        dx[:, t] = e * (1 - a[:, t])
        dg[:, t] = e * (every[:, t] - x[:, t]) * a[:, t] * (1 - a[:, t])
        e = e * a[:, t]
    return dg, dx, e
