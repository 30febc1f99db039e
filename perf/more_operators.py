"""Measured calls of the operators that train a model's head: layer norm, activations kept in 8 bits, and the loss over a vocabulary.

  norm       layer norm of rows (an inference call: nothing is kept)
  norm_step  a training step's two calls: the layer norm, which keeps its input in 8 bits, and the gradients from those 8 bits
  norm_grad  the gradients from the input as it was
  loss       softmax cross entropy of x W^T against a class a row, without logits in memory (scoring, evaluation)
  loss_step  a training step's two calls: the loss, which keeps two numbers a row, and the gradients of x and W
  weight     gradient of a dense layer's weights from the layer's input as 8-bit rows, with the bias's gradient

Rows are tokens, or the nodes or graphs of a batch.  Everything is made on the GPU from the seed.
"""
from __future__ import annotations

import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_EPS = 1e-5
_STREAM = None
_CONTEXT = None


def listed():
    return [
        # a mini-batch of graph embeddings in front of the readout: launches and host work are everything
        _norm("norm_graphs_64", "norm", 64, 128, "f32"),
        # one layer's training step over the tokens of a batch, the input kept in a byte an element
        _norm("norm_step_tokens_8k", "norm_step", 8192, 8192, "bf16"),
        # an odd width: no row but the first is aligned
        _norm("norm_step_ragged", "norm_step", 1531, 1021, "f16"),
        # the node embeddings of the large molecule batch (16,384 graphs, d = 128): short rows, a long sum for the weight's gradient
        _norm("norm_grad_nodes", "norm_grad", 491520, 128, "f32"),
        # one token scored against a vocabulary: W is read once
        _loss("loss_one_token", "loss", 1, 131072, 4096, "bf16"),
        # an evaluation batch
        _loss("loss_vocab_128k", "loss", 4096, 131072, 2048, "bf16"),
        # a graph classifier's mini-batch
        _loss("loss_step_graphs_64", "loss_step", 64, 6, 128, "f32"),
        # the same model's largest batch, more classes
        _loss("loss_step_classes_f32", "loss_step", 16384, 1000, 256, "f32"),
        # nothing a multiple of a tile, rows at odd places, a small vocabulary
        _loss("loss_step_ragged", "loss_step", 1531, 50021, 1021, "f16"),
        # a language model's training step
        _loss("loss_step_vocab_128k", "loss_step", 4096, 131072, 4096, "bf16"),
        # a wide layer of a long batch
        _weight("weight_8k", 8192, 4096, 4096, "bf16"),
        # the hidden layer of the large molecule batch: a small result summed over many nodes
        _weight("weight_nodes", 491520, 256, 128, "f32"),
    ]


def draw(rng):
    """One more case; sizes log-uniform, odd ones among them, none that costs more than the largest listed one of its kind."""
    kind = rng.choice(["norm", "norm_step", "norm_grad", "loss", "loss_step", "loss_step", "weight", "weight"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if kind.startswith("norm"):
        cols = _log_int(rng, 8, 16384)
        return _norm(None, kind, _log_int(rng, 1, min(1 << 19, (1 << 26) * 2 // _BYTES[dtype] // cols)), cols, dtype)
    if kind == "weight":
        n, k = _log_int(rng, 2, 14336), _log_int(rng, 8, 14336)
        most = min(1 << 19, (1 << 27) // max(n, k), (1 << 37) // (n * k))
        return _weight(None, _log_int(rng, 1, max(1, most)), n, k, dtype)
    vocab, k = rng.choice([rng.randint(2, 40), _log_int(rng, 40, 4096), _log_int(rng, 4096, 200000), _log_int(rng, 4096, 200000)]), _log_int(rng, 16, 8192)
    most = min(16384, (1 << 39) // (vocab * k), (1 << 30) // vocab, (1 << 27) // k)
    return _loss(None, kind, _log_int(rng, 1, max(1, most)), vocab, k, dtype)


def prepare(case, seed):
    global _STREAM
    if _STREAM is None:
        _STREAM = torch.cuda.Stream()
    torch.cuda.set_stream(_STREAM)   # one stream for the library's work and torch's allocations, as in a user's loop
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 7919 + 29)
    kind, dtype = case["kind"], _TYPES[case["dtype"]]
    # gradients of 16 bits with a small range of exponents are scaled up, as training in that type does
    loss_scale = 8192.0 if case["dtype"] == "f16" else 1.0
    if kind.startswith("norm"):
        rows, cols = case["rows"], case["cols"]
        state = {"case": case, "x": _activations(rows, cols, dtype, gen), "weight": 1.0 + 0.2 * torch.randn(cols, generator=gen, device="cuda"),
                 "bias": 0.1 * torch.randn(cols, generator=gen, device="cuda")}
        if kind != "norm":
            state["dy"] = (torch.randn((rows, cols), generator=gen, device="cuda") * (loss_scale / 4096)).to(dtype)
        if kind == "norm_grad":
            state["stats"] = _moments(state["x"].double()).float()
        return state
    if kind == "weight":
        m, n, k = case["m"], case["n"], case["k"]
        q, scale = _integers(_activations(m, k, torch.float32, gen))
        dy = torch.randn((m, n), generator=gen, device="cuda") * (loss_scale / 4096)
        dy *= 0.25 + torch.rand((m, 1), generator=gen, device="cuda")
        return {"case": case, "dy": dy.to(dtype), "q": _pitched(q), "scale": scale}
    rows, vocab, k = case["rows"], case["vocab"], case["k"]
    W = (torch.randn((vocab, k), generator=gen, device="cuda") * (2.0 / math.sqrt(k))).to(dtype)
    # small indices are likelier, as words are
    target = (vocab ** torch.rand(rows, generator=gen, device="cuda")).long().clamp(1, vocab) - 1
    x = torch.randn((rows, k), generator=gen, device="cuda")
    x += (2.5 * torch.rand((rows, 1), generator=gen, device="cuda")) * W[target].float()   # some rows know their class, some don't
    if rows > 1:   # padding: no class, and nothing in the row
        padded = torch.rand(rows, generator=gen, device="cuda") < 0.05
        target[padded] = -1
        x[padded] = 0.0
    weight = torch.full((rows,), loss_scale / max(1, int((target >= 0).sum())), device="cuda")   # the mean over the rows that count
    return {"case": case, "x": x.to(dtype), "W": W, "target": target.to(torch.int32), "weight": weight}


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        return _own(state, case, kind)
    if kind == "norm":
        return {"y": _normed(state, _moments(state["x"].float()))}
    if kind == "norm_step":
        x = state["x"].float()
        moments = _moments(x)
        q, scale = _integers(x)
        return {"y": _normed(state, moments), **_norm_gradients(state, q.float() * scale[:, None], moments)}
    if kind == "norm_grad":
        return _norm_gradients(state, state["x"].float(), state["stats"])
    if kind == "weight":
        dy = state["dy"].float()
        x = state["q"].float() * state["scale"][:, None]
        return {"dW": (dy.t() @ x).to(_TYPES[case["dtype"]]), "dbias": dy.sum(dim=0, dtype=torch.float64).float()}
    return _plain_loss(state, case)


def work(case):
    kind, es = case["kind"], _BYTES[case["dtype"]]
    if kind.startswith("norm"):
        rows, cols = case["rows"], case["cols"]
        n = rows * cols
        if kind == "norm":
            return {"bytes": 2 * n * es + 8 * cols, "flops": 8 * n}
        if kind == "norm_grad":   # x and dy read, dx written
            return {"bytes": 3 * n * es + 8 * rows + 12 * cols, "flops": 14 * n}
        # x read, y and the 8-bit rows written; then those and dy read, dx written
        return {"bytes": n * (4 * es + 2) + 24 * rows + 20 * cols, "flops": 25 * n}
    if kind == "weight":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * n * es + m * k + 4 * m + n * k * es + 4 * n, "flops": 2 * m * n * k}
    rows, vocab, k = case["rows"], case["vocab"], case["k"]
    if kind == "loss":
        return {"bytes": (rows + vocab) * k * es + 12 * rows, "flops": 2 * rows * vocab * k}
    # the loss, and then, without kept logits, these again and the two gradients' products
    return {"bytes": 3 * (rows + vocab) * k * es + 28 * rows, "flops": 8 * rows * vocab * k}


def exact(case, seed):
    """The same from the definitions in 64 bits.  The 8-bit rows are part of the definition: the integers nearest to x * r as fp32 has it, r = 127 / max |x|."""
    state = prepare(case, seed)
    kind = case["kind"]
    if kind.startswith("norm"):
        x = state["x"].double()
        if kind == "norm_grad":
            mean, rstd = state["stats"].double().unbind(1)
        else:
            var, mean = torch.var_mean(x, dim=1, correction=0)
            rstd = 1.0 / torch.sqrt(var + _EPS)
        gamma = state["weight"].double()
        out = {}
        if kind != "norm_grad":
            out["y"] = (x - mean[:, None]) * rstd[:, None] * gamma + state["bias"].double()
        if kind == "norm":
            return out
        if kind == "norm_step":   # a product of two fp32 values is exact in 64 bits; the scale is the one kept, in fp32
            biggest = x.abs().amax(dim=1)
            x = (x * torch.where(biggest > 0, 127.0 / biggest, 0.0).float().double()[:, None]).float().double().round() * (biggest / 127.0).float().double()[:, None]
        hat = (x - mean[:, None]) * rstd[:, None]
        dy = state["dy"].double()
        g = dy * gamma
        out["dx"] = rstd[:, None] * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
        out["dweight"], out["dbias"] = (dy * hat).sum(0), dy.sum(0)
        return out
    if kind == "weight":
        m, n, k = case["m"], case["n"], case["k"]
        dW = torch.zeros((n, k), dtype=torch.float64, device="cuda")
        dbias = torch.zeros(n, dtype=torch.float64, device="cuda")
        step = max(1, (1 << 27) // max(n, k))
        for a in range(0, m, step):
            dy = state["dy"][a:a + step].double()
            dW += dy.t() @ (state["q"][a:a + step].double() * state["scale"][a:a + step, None].double())
            dbias += dy.sum(0)
        return {"dW": dW, "dbias": dbias}
    rows, vocab, k = case["rows"], case["vocab"], case["k"]
    W, loss = state["W"].double(), torch.zeros(rows, dtype=torch.float64, device="cuda")
    dx, dW = torch.zeros((rows, k), dtype=torch.float64, device="cuda"), torch.zeros((vocab, k), dtype=torch.float64, device="cuda")
    step = max(1, (1 << 27) // vocab)
    for a in range(0, rows, step):
        at = slice(a, min(rows, a + step))
        x, t = state["x"][at].double(), state["target"][at].long()
        counts = (t >= 0) & (t < vocab)
        w = torch.where(counts, state["weight"][at].double(), 0.0)
        z = x @ W.t()
        lse = torch.logsumexp(z, dim=1)
        mine = z.gather(1, t.clamp(0, vocab - 1)[:, None])[:, 0]
        loss[at] = w * (lse - mine)
        if kind == "loss_step":
            z = (z - lse[:, None]).exp()
            z.scatter_add_(1, t.clamp(0, vocab - 1)[:, None], torch.full((z.shape[0], 1), -1.0, dtype=torch.float64, device="cuda"))
            z *= w[:, None]
            dx[at] = z @ W
            dW += z.t() @ x
    return {"loss": loss, "dx": dx, "dW": dW} if kind == "loss_step" else {"loss": loss}


# ---------------------------------------------------------------- the framework's calls
def _own(state, case, kind):
    ctx, stream = _context(), torch.cuda.current_stream().cuda_stream
    if kind.startswith("norm"):
        x, rows, cols = state["x"], case["rows"], case["cols"]
        out = {}
        if kind == "norm":
            out["y"] = torch.empty_like(x)
            ctx.layer_norm(x, out["y"], weight=state["weight"], bias=state["bias"], eps=_EPS, stream=stream)
            return out
        if "workspace" not in state:
            state["workspace"] = _bytes(ctx.layer_norm_grad_workspace_bytes(rows, cols))
        out.update(dx=torch.empty_like(x), dweight=torch.empty(cols, device="cuda"), dbias=torch.empty(cols, device="cuda"))
        if kind == "norm_grad":
            ctx.layer_norm_grad(state["dy"], state["stats"], out["dx"], state["workspace"], x=x, weight=state["weight"], dweight=out["dweight"], dbias=out["dbias"], stream=stream)
            return out
        out["y"], stats = torch.empty_like(x), torch.empty((rows, 2), device="cuda")
        q, scale = torch.empty((rows, cols), dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
        ctx.layer_norm(x, out["y"], weight=state["weight"], bias=state["bias"], eps=_EPS, stats=stats, q=q, q_scale=scale, stream=stream)
        ctx.layer_norm_grad(state["dy"], stats, out["dx"], state["workspace"], q=q, q_scale=scale, weight=state["weight"], dweight=out["dweight"], dbias=out["dbias"], stream=stream)
        return out
    if kind == "weight":
        m, n, k = case["m"], case["n"], case["k"]
        if "workspace" not in state:
            state["workspace"] = _bytes(ctx.linear_i8_grad_workspace_bytes(m, n, k, _TYPES[case["dtype"]]))
        dW, dbias = torch.empty((n, k), dtype=_TYPES[case["dtype"]], device="cuda"), torch.empty(n, device="cuda")
        ctx.linear_i8_grad(state["dy"], state["q"], state["scale"], dW, state["workspace"], dbias=dbias, stream=stream)
        return {"dW": dW, "dbias": dbias}
    x, W, target, weight = state["x"], state["W"], state["target"], state["weight"]
    rows, vocab, k = case["rows"], case["vocab"], case["k"]
    if "workspace" not in state:
        state["workspace"] = _bytes(ctx.linear_cross_entropy_workspace_bytes(rows, vocab, k, _TYPES[case["dtype"]], grad=kind == "loss_step"))
    loss = torch.empty(rows, device="cuda")
    if kind == "loss":
        ctx.linear_cross_entropy(x, W, target, loss, state["workspace"], row_weight=weight, stream=stream)
        return {"loss": loss}
    stats, dx, dW = torch.empty((rows, 2), device="cuda"), torch.empty_like(x), torch.empty_like(W)
    ctx.linear_cross_entropy(x, W, target, loss, state["workspace"], row_weight=weight, stats=stats, stream=stream)
    ctx.linear_cross_entropy_grad(x, W, target, stats, state["workspace"], dx=dx, dW=dW, row_weight=weight, stream=stream)
    return {"loss": loss, "dx": dx, "dW": dW}


def _context():
    global _CONTEXT
    if _CONTEXT is None:
        from graphnn_b200 import capi
        _CONTEXT = capi.Context(0)
    return _CONTEXT


def _bytes(n):
    return torch.empty(n, dtype=torch.uint8, device="cuda")


# ---------------------------------------------------------------- the plain forms
def _moments(x):
    """Mean and 1 / deviation of each row, [rows x 2], in the type of x."""
    mean = x.mean(dim=1)
    var = (x - mean[:, None]).square().mean(dim=1)
    return torch.stack([mean, 1.0 / (var + _EPS).sqrt()], dim=1)


def _normed(state, moments):
    x = state["x"].float()
    return ((x - moments[:, :1]) * moments[:, 1:] * state["weight"] + state["bias"]).to(state["x"].dtype)


def _norm_gradients(state, x, moments):
    hat = (x - moments[:, :1]) * moments[:, 1:]
    dy = state["dy"].float()
    g = dy * state["weight"]
    dx = moments[:, 1:] * (g - g.mean(dim=1, keepdim=True) - hat * (g * hat).mean(dim=1, keepdim=True))
    return {"dx": dx.to(state["x"].dtype), "dweight": (dy * hat).sum(dim=0, dtype=torch.float64).float(), "dbias": dy.sum(dim=0, dtype=torch.float64).float()}


def _plain_loss(state, case):
    rows, vocab, k, dtype = case["rows"], case["vocab"], case["k"], _TYPES[case["dtype"]]
    step = max(1, (1 << 28) // vocab)
    W = state["W"].float()
    loss = torch.empty(rows, device="cuda")
    dx = torch.empty((rows, k), device="cuda")
    dW = None
    for a in range(0, rows, step):
        at = slice(a, min(rows, a + step))
        x, t = state["x"][at].float(), state["target"][at].long()
        counts = (t >= 0) & (t < vocab)
        where = torch.where(counts, t, 0)[:, None]
        w = torch.where(counts, state["weight"][at], 0.0)
        z = x @ W.t()
        z = z - z.gather(1, where)                       # against the row's own class, whose share of the sum is then exactly 1
        z.scatter_(1, where, float("-inf"))
        top = z.amax(dim=1).clamp(min=0)
        others = (z - top[:, None]).exp().sum(dim=1)
        one = torch.where(top > 0, top + (others + (-top).exp()).log(), torch.log1p(others))
        loss[at] = one * w
        if case["kind"] == "loss":
            continue
        g = (z - one[:, None]).exp()
        g.scatter_(1, where, torch.expm1(-one)[:, None])
        g = g * w[:, None]
        dx[at] = g @ W
        dW = g.t() @ x if dW is None else dW + g.t() @ x
    if case["kind"] == "loss":
        return {"loss": loss}
    return {"loss": loss, "dx": dx.to(dtype), "dW": dW.to(dtype)}


# ---------------------------------------------------------------- inputs
def _integers(x):
    """Rows in fp32 -> 8-bit integers and a scale for each row."""
    biggest = x.abs().amax(dim=1)
    limit = torch.full((), 127.0, device=x.device)   # a tensor: torch replaces the division by a number with a product
    factor = torch.where(biggest >= 2.0 ** -110, limit / biggest, 0.0)
    return (x * factor[:, None]).round().to(torch.int8), torch.where(biggest >= 2.0 ** -110, biggest / limit, 0.0)


def _activations(rows, cols, dtype, gen):
    """Rows of different sizes and means, and a few channels that stand out, as activations have them."""
    x = torch.randn((rows, cols), generator=gen, device="cuda")
    x *= torch.where(torch.rand(cols, generator=gen, device="cuda") < 0.01, 8.0, 1.0)
    x *= 0.5 + torch.rand((rows, 1), generator=gen, device="cuda")
    x += 0.5 * torch.randn((rows, 1), generator=gen, device="cuda")
    return x.to(dtype)


def _pitched(q):
    """The rows of an 8-bit matrix on 16-byte boundaries, as the 8-bit products want them too."""
    rows, cols = q.shape
    if cols % 16 == 0:
        return q
    wide = torch.zeros((rows, (cols + 15) // 16 * 16), dtype=q.dtype, device="cuda")
    wide[:, :cols] = q
    return wide[:, :cols]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _norm(name, kind, rows, cols, dtype):
    case = {"kind": kind, "rows": rows, "cols": cols, "dtype": dtype}
    return dict(case, name=name) if name else case


def _loss(name, kind, rows, vocab, k, dtype):
    case = {"kind": kind, "rows": rows, "vocab": vocab, "k": k, "dtype": dtype}
    return dict(case, name=name) if name else case


def _weight(name, m, n, k, dtype):
    case = {"kind": "weight", "m": m, "n": n, "k": k, "dtype": dtype}
    return dict(case, name=name) if name else case
