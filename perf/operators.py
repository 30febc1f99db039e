"""Measured calls of the operators for compressed models: products in 8-bit integers and distillation from a teacher's top logits.

  quantize  rows of activations (or of a weight matrix, a channel a row) to 8-bit integers with a scale for each row
  gemm      product of two such matrices, scales for each token and channel, bias and ReLU in the same pass
  linear    the layer as a model runs it: activations in their own type, 8-bit weights, output in the activations' type
  distill   Kullback-Leibler loss of a student's logits against the top logits of a teacher, with its gradient in the same call
  distill2  the same as two calls: the loss, which keeps each row's statistics, and later the gradient

Rows are tokens, or the nodes or graphs of a batch.  Everything is made on the GPU from the seed.
"""
from __future__ import annotations

import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_STREAM = None
_CONTEXT = None


def listed():
    return [
        # a handful of graph embeddings on their way into the readout: launches and host work are everything
        _quantize("quantize_graphs_64", 64, 128, "f32"),
        # the activations of a long prompt
        _quantize("quantize_tokens_8k", 8192, 8192, "bf16"),
        # nothing a multiple of a tile, output kept in fp32 for a following reduction
        _gemm("gemm_ragged", 333, 1021, 1504, "f32", bias=True, relu=False),
        # an ordinary layer over a few thousand tokens
        _gemm("gemm_4k", 4096, 4096, 4096, "bf16", bias=False, relu=False),
        # the largest products: a wide layer over a long batch
        _gemm("gemm_8k", 8192, 8192, 8192, "bf16", bias=False, relu=False),
        # one token of a serving loop
        _linear("linear_one_token", 1, 4096, 4096, "bf16", bias=False, relu=False),
        # a few dozen sequences that each ask for their next token
        _linear("linear_27_tokens", 27, 14336, 4096, "f16", bias=True, relu=False),
        # the node embeddings of the large molecule batch (16,384 graphs, d = 128) through a hidden layer of 256
        _linear("linear_nodes", 491520, 256, 128, "f32", bias=True, relu=True),
        # a classifier's mini-batch, half of the classes in the teacher's list, the teacher's full normaliser known
        _distill("distill_graphs_64", "distill", 64, 6, 3, "f32", 2.0, tail=True),
        # a language model's batch: long rows, every logit read and every gradient written once
        _distill("distill_vocab_128k", "distill", 4096, 131072, 64, "bf16", 1.0, tail=True),
        # loss and gradient as two calls, an odd vocabulary: no row but the first is aligned
        _distill("distill_two_calls_50k", "distill2", 1531, 50021, 50, "f16", 1.5, tail=False),
        # few long rows in fp32: one sequence being looked at
        _distill("distill_two_calls_24_rows", "distill2", 24, 151000, 128, "f32", 1.0, tail=True),
    ]


def draw(rng):
    """One more case; sizes log-uniform, odd ones among them, none that costs more than the largest listed one of its kind."""
    kind = rng.choice(["quantize", "quantize", "gemm", "gemm", "gemm", "linear", "linear", "linear", "distill", "distill", "distill2", "distill2"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if kind == "quantize":
        cols = _log_int(rng, 8, 16384)
        return _quantize(None, _log_int(rng, 1, min(1 << 19, (1 << 26) * 2 // _BYTES[dtype] // cols)), cols, dtype)
    if kind == "gemm":
        n, k = _log_int(rng, 16, 14336), _log_int(rng, 32, 14336)
        return _gemm(None, _log_int(rng, 1, min(16384, (1 << 38) // (n * k))), n, k, dtype, bias=rng.random() < 0.5, relu=rng.random() < 0.3)
    if kind == "linear":
        n, k = _log_int(rng, 16, 14336), _log_int(rng, 32, 14336)
        most = min(1 << 19, (1 << 27) // max(n, k), (1 << 37) // (n * k))
        return _linear(None, _log_int(rng, 1, rng.choice([1, 8, 64, most, most])), n, k, dtype, bias=rng.random() < 0.5, relu=rng.random() < 0.3)
    cols = rng.choice([rng.randint(2, 40), _log_int(rng, 32, 4096), _log_int(rng, 4096, 200000), _log_int(rng, 4096, 200000)])
    rows = _log_int(rng, 1, min(16384, (1 << 28) // cols))
    return _distill(None, kind, rows, cols, min(cols, _log_int(rng, 1, 128)), dtype, rng.choice([1.0, 1.0, 2.0, 0.5, 4.0]), tail=rng.random() < 0.5)


def prepare(case, seed):
    global _STREAM
    if _STREAM is None:
        _STREAM = torch.cuda.Stream()
    torch.cuda.set_stream(_STREAM)   # one stream for the library's work and torch's allocations, as in a user's loop
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 6151 + 17)
    kind, dtype = case["kind"], _TYPES[case["dtype"]]
    if kind == "quantize":
        return {"case": case, "x": _activations(case["rows"], case["cols"], dtype, gen)}
    if kind in ("gemm", "linear"):
        m, n, k = case["m"], case["n"], case["k"]
        w, w_scale = _integers(torch.randn((n, k), generator=gen, device="cuda") / math.sqrt(k))
        state = {"case": case, "w": _pitched(w), "w_scale": w_scale, "bias": torch.randn(n, generator=gen, device="cuda") * 0.1 if case["bias"] else None}
        x = _activations(m, k, dtype, gen)
        if kind == "gemm":
            q, scale = _integers(x.float())
            state.update(x=_pitched(q), x_scale=scale)
        else:
            state.update(x=x)
        return state
    rows, cols, top = case["rows"], case["cols"], case["top"]
    prior = 2.0 * torch.randn(cols, generator=gen, device="cuda")   # some classes are likelier than others in every row
    z = torch.empty((rows, cols), dtype=dtype, device="cuda")
    idx = torch.empty((rows, top), dtype=torch.int32, device="cuda")
    t = torch.empty((rows, top), dtype=torch.float32, device="cuda")
    lse = torch.empty(rows, dtype=torch.float32, device="cuda")
    step = max(1, (1 << 27) // cols)
    for a in range(0, rows, step):
        b = min(rows, a + step)
        teacher = prior + 2.0 * torch.randn((b - a, cols), generator=gen, device="cuda")
        z[a:b] = (0.8 * teacher + 0.8 * torch.randn((b - a, cols), generator=gen, device="cuda")).to(dtype)
        t[a:b], i = torch.topk(teacher, top, dim=1)
        idx[a:b] = i.to(torch.int32)
        lse[a:b] = torch.logsumexp(teacher.double() / case["temperature"], 1).float() if cols <= 4096 else torch.logsumexp(teacher / case["temperature"], 1)
    # some lists are shorter (a nucleus instead of a fixed count: -1 behind the last), and padded rows have none and no weight
    kept = torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.2, 1 + (torch.rand(rows, generator=gen, device="cuda") * top).long(), top)
    kept = torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.03, 0, kept)
    idx[torch.arange(top, device="cuda")[None, :] >= kept[:, None]] = -1
    # the mean over the rows that count; gradients of 16 bits with a small range of exponents are scaled up, as training in that type does
    weight = (kept > 0).float() * ((8192.0 if case["dtype"] == "f16" else 1.0) / max(1, int((kept > 0).sum())))
    return {"case": case, "z": z, "idx": idx, "t": t, "t_lse": lse if case["tail"] else None, "weight": weight}


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        ctx, stream = _context(), torch.cuda.current_stream().cuda_stream
        if kind == "quantize":
            x = state["x"]
            q, scale = torch.empty(x.shape, dtype=torch.int8, device="cuda"), torch.empty(x.shape[0], device="cuda")
            ctx.quantize_rows_i8(x, q, scale, stream=stream)
            return {"q": q, "scale": scale}
        if kind == "gemm":
            out = torch.empty((case["m"], case["n"]), dtype=_TYPES[case["dtype"]], device="cuda")
            ctx.gemm_i8(state["x"], state["x_scale"], state["w"], state["w_scale"], out, bias=state["bias"], relu=case["relu"], stream=stream)
            return {"y": out}
        if kind == "linear":
            if "workspace" not in state:
                state["workspace"] = torch.empty(ctx.linear_i8_workspace_bytes(case["m"], case["k"]), dtype=torch.uint8, device="cuda")
            out = torch.empty((case["m"], case["n"]), dtype=_TYPES[case["dtype"]], device="cuda")
            ctx.linear_i8(state["x"], state["w"], state["w_scale"], out, state["workspace"], bias=state["bias"], relu=case["relu"], stream=stream)
            return {"y": out}
        z = state["z"]
        loss, dz = torch.empty(z.shape[0], device="cuda"), torch.empty_like(z)
        more = {"temperature": case["temperature"], "t_lse": state["t_lse"], "row_weight": state["weight"], "stream": stream}
        if kind == "distill":
            ctx.distill_topk(z, state["idx"], state["t"], loss, dz=dz, **more)
        else:
            stats = torch.empty((z.shape[0], 4), device="cuda")
            ctx.distill_topk(z, state["idx"], state["t"], loss, stats=stats, **more)
            ctx.distill_topk_grad(z, state["idx"], state["t"], stats, dz, **more)
        return {"loss": loss, "dz": dz}
    if kind == "quantize":
        q, scale = _integers(state["x"].float())
        return {"q": q, "scale": scale}
    if kind == "gemm":
        return {"y": _product(case, state, state["x"], state["x_scale"])}
    if kind == "linear":
        return {"y": _product(case, state, *_integers(state["x"].float()))}
    return _distillation(case, state)


def work(case):
    kind, es = case["kind"], _BYTES[case["dtype"]]
    if kind == "quantize":
        rows, cols = case["rows"], case["cols"]
        return {"bytes": rows * cols * (es + 1) + 4 * rows, "flops": 3 * rows * cols}
    if kind in ("gemm", "linear"):
        m, n, k = case["m"], case["n"], case["k"]
        x = m * k * es if kind == "linear" else m * k + 4 * m
        return {"bytes": x + n * k + 4 * n * (2 if case["bias"] else 1) + m * n * es, "flops": 2 * m * n * k}
    rows, cols, top = case["rows"], case["cols"], case["top"]
    # the logits read once, the gradient written once, the teacher's lists, weight and loss (and normaliser) of each row
    return {"bytes": 2 * rows * cols * es + rows * (8 * top + (12 if case["tail"] else 8)), "flops": 8 * rows * cols}


def exact(case, seed):
    """The same from the definitions in 64 bits.  The 8-bit integers are part of the definition: the nearest to x * r as fp32 has it, r = 127 / max |x|."""
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        biggest = state["x"].double().abs().max(dim=1).values
        return {"q": None, "scale": biggest / 127.0}   # whole numbers are compared as they are
    if kind in ("gemm", "linear"):
        if kind == "gemm":
            q, scale = state["x"].double(), state["x_scale"].double()
        else:
            x = state["x"].double()
            biggest = x.abs().max(dim=1).values
            factor = torch.where(biggest > 0, 127.0 / biggest, 0.0).float().double()
            q, scale = (x * factor[:, None]).float().double().round(), biggest / 127.0   # a product of two fp32 values is exact in 64 bits
        out = torch.empty((case["m"], case["n"]), dtype=torch.float64, device="cuda")
        w = state["w"].double().t()
        step = max(1, (1 << 28) // max(case["n"], case["k"]))
        for a in range(0, case["m"], step):
            y = (q[a:a + step] @ w) * scale[a:a + step, None] * state["w_scale"].double()
            if state["bias"] is not None:
                y += state["bias"].double()
            out[a:a + step] = y.clamp(min=0) if case["relu"] else y
        return {"y": out}
    rows, cols, temp = case["rows"], case["cols"], case["temperature"]
    loss = torch.zeros(rows, dtype=torch.float64, device="cuda")
    dz = torch.zeros((rows, cols), dtype=torch.float64, device="cuda")
    step = max(1, (1 << 26) // cols)
    for a in range(0, rows, step):
        at = slice(a, min(rows, a + step))
        valid = state["idx"][at] >= 0
        some = valid.any(dim=1)
        where = torch.where(valid, state["idx"][at], 0).long()
        scaled = torch.where(valid, state["t"][at].double() / temp, float("-inf"))
        if case["tail"]:
            p = (scaled - state["t_lse"][at].double()[:, None]).exp()
        else:
            p = torch.where(some[:, None], scaled, 0.0).softmax(dim=1)
        log_q = (state["z"][at].double() / temp).log_softmax(dim=1)
        target = torch.zeros_like(log_q).scatter_add_(1, where, torch.where(valid, p, 0.0))
        kl = torch.where(valid & (p > 0), p * (p.log() - log_q.gather(1, where)), 0.0).sum(dim=1)
        grad = log_q.exp() - target
        if case["tail"]:
            inside = torch.zeros_like(log_q).scatter_add_(1, where, valid.double()) > 0
            rest = (1.0 - torch.where(valid, p, 0.0).sum(dim=1)).clamp(min=0)
            out_q = log_q.masked_fill(inside, float("-inf"))
            log_s = out_q.logsumexp(dim=1)
            kl += torch.where((rest > 0) & (log_s > float("-inf")), rest * (rest.log() - log_s), 0.0)
            grad -= torch.where(log_s > float("-inf"), rest, 0.0)[:, None] * (out_q - torch.where(log_s > float("-inf"), log_s, 0.0)[:, None]).exp()
        w = state["weight"][at].double()
        loss[at] = torch.where(some, kl * w, 0.0)
        dz[at] = torch.where(some[:, None], grad * (w / temp)[:, None], 0.0)
    return {"loss": loss, "dz": dz}


# ---------------------------------------------------------------- the plain forms
def _integers(x):
    """Rows in fp32 -> 8-bit integers and a scale for each row."""
    biggest = x.abs().amax(dim=1)
    limit = torch.full((), 127.0, device=x.device)   # a tensor: torch replaces the division by a number with a product
    factor = torch.where(biggest >= 2.0 ** -110, limit / biggest, 0.0)
    return (x * factor[:, None]).round().to(torch.int8), torch.where(biggest >= 2.0 ** -110, biggest / limit, 0.0)


def _product(case, state, q, scale):
    y = (q.float() @ state["w"].float().t()) * (scale[:, None] * state["w_scale"][None, :])
    if state["bias"] is not None:
        y = y + state["bias"]
    if case["relu"]:
        y = torch.where(y < 0, 0.0, y)
    return y.to(_TYPES[case["dtype"]])


def _distillation(case, state):
    temp = case["temperature"]
    z = state["z"].float() / temp
    top = z.amax(dim=1, keepdim=True)
    e = (z - top).exp()
    valid = state["idx"] >= 0
    where = state["idx"].clamp(min=0).long()
    # what is per row and per entry of the lists: in 64 bits, for the small masses on either side of a list
    scaled = torch.where(valid, state["t"].double() / temp, float("-inf"))
    if case["tail"]:
        p = (scaled - state["t_lse"].double()[:, None]).exp()
        outside = torch.zeros_like(z).scatter_add_(1, where, valid.float()) == 0
        tail = torch.where(outside, e, 0.0).sum(dim=1).double()
        listed_part = torch.where(valid, e.gather(1, where).double(), 0.0).sum(dim=1)
        total = tail + listed_part
    else:
        p = (scaled - scaled.amax(dim=1, keepdim=True)).exp()
        p = p / p.sum(dim=1, keepdim=True)
        total = e.sum(dim=1).double()
    p = torch.where(valid, p, 0.0)   # also where the whole list is empty
    log_q = (z.gather(1, where) - top).double() - total.log()[:, None]
    loss = torch.where(p > 0, p * (p.log() - log_q), 0.0).sum(dim=1)
    weight = torch.where(valid.any(dim=1), state["weight"], 0.0)
    grad = e / total.float()[:, None]
    if case["tail"]:
        given = p.sum(dim=1)
        rest = (1.0 - given).clamp(min=0)
        loss = loss + torch.where((rest > 0) & (tail > 0), rest * (torch.log1p(-given.clamp(max=1.0)) + torch.log1p(listed_part / tail)), 0.0)
        keep = torch.where(tail > 0, 1.0 - rest * total / tail, 0.0).float()
        grad = torch.where(outside, grad * keep[:, None], grad)
    grad = grad.scatter_add_(1, where, -p.float()) * (weight / temp)[:, None]
    return {"loss": (loss * weight).float(), "dz": grad.to(state["z"].dtype)}


# ---------------------------------------------------------------- inputs
def _context():
    global _CONTEXT
    if _CONTEXT is None:
        from graphnn_b200 import capi
        _CONTEXT = capi.Context(0)
    return _CONTEXT


def _activations(rows, cols, dtype, gen):
    """Rows of different sizes, and a few channels that stand out, as activations have them."""
    x = torch.randn((rows, cols), generator=gen, device="cuda")
    x *= torch.where(torch.rand(cols, generator=gen, device="cuda") < 0.01, 8.0, 1.0)
    x *= 0.5 + torch.rand((rows, 1), generator=gen, device="cuda")
    return x.to(dtype)


def _pitched(q):
    """The rows of an 8-bit matrix on 16-byte boundaries, where the product wants them."""
    rows, cols = q.shape
    if cols % 16 == 0:
        return q
    wide = torch.zeros((rows, (cols + 15) // 16 * 16), dtype=q.dtype, device="cuda")
    wide[:, :cols] = q
    return wide[:, :cols]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _quantize(name, rows, cols, dtype):
    case = {"kind": "quantize", "rows": rows, "cols": cols, "dtype": dtype}
    return dict(case, name=name) if name else case


def _gemm(name, m, n, k, dtype, bias, relu):
    case = {"kind": "gemm", "m": m, "n": n, "k": k, "dtype": dtype, "bias": bias, "relu": relu}
    return dict(case, name=name) if name else case


def _linear(name, m, n, k, dtype, bias, relu):
    return dict(_gemm(name, m, n, k, dtype, bias, relu), kind="linear")


def _distill(name, kind, rows, cols, top, dtype, temperature, tail):
    case = {"kind": kind, "rows": rows, "cols": cols, "top": top, "dtype": dtype, "temperature": temperature, "tail": tail}
    return dict(case, name=name) if name else case
